"""The paged K/V cache (write, read, attention) and cross attention on the GPU,
against oracle/paged.py in float64.

Tolerances, from the arithmetic:
  * codes, scales: the codes equal the exact quotient's (paged_kv.cu says why);
    scale = a / Q rounded once, 2^-24 relative;
  * read back: code * scale in f32 rounded to bf16, 2^-8 relative, plus 2^-24;
  * attention: with A = sum p |v| / sum p of a row's output,
      2^-8 A   each p is rounded to bf16 for the matrix instruction,
      2^-8 |o| the output is rounded to bf16,
      5e-4 A   both exponentials' polynomial (7.5e-5, in p and in the sum), f32
               scores of at most 128 products, f32 sums;
    over 8-bit pages p and code * scale are rounded to f16, half a step of which
    is 2^-11: 2^-11 A more for v, and for k each score moves by at most
    d = 2^-11 sum_i |q_i k_i| / sqrt(128), so each p, and each sum of p, by a
    factor within exp(+-d): exp(2 d) - 1 of A more;
  * lse: 2e-4 for the polynomial in the sum, f32 rounding of the value, and d.
"""

import math

import pytest
import torch

from oracle import paged as O

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]

DEV = "cuda"
BF, E4, S8 = torch.bfloat16, torch.uint8, torch.int8
DTYPES = [BF, E4, S8]
SCALE = 128 ** -0.5


def K():
    from waveforcing_b200 import kernels

    return kernels


def healthy():
    from waveforcing_b200 import _lib

    assert _lib.status_take() == 0


def most_move(q, k):
    """d of the header: q [.., n, 128] against k [.., L, 128] of the same heads."""
    return 2 ** -11 * SCALE * float((q.double().abs() @ k.nan_to_num(0.0).double().abs().transpose(-1, -2)).max())


def score_move(pool, q):
    if pool.dtype == BF:
        return 0.0
    k = pool.val[0].transpose(0, 1).flatten(1, 2)  # [heads, keys, 128]
    return most_move(q.transpose(0, 1), k.repeat_interleave(q.shape[1] // k.shape[0], 0))


class Pool:
    """A CPU pool whose rows hold garbage (NaN values, NaN scales) wherever no
    sequence has a position, its f64 values, and its copy on the GPU."""

    def __init__(self, dtype, lens, heads, ps, seed, spare=2, token_major=False, max_pages=None):
        g = torch.Generator().manual_seed(seed)
        need = [-(-t // ps) for t in lens]
        P = sum(need) + spare
        order = torch.randperm(P, generator=g).tolist()
        width = max_pages or max([1] + need)
        self.table, self.ps, self.heads, self.P, self.lens, self.dtype = [], ps, heads, P, list(lens), dtype
        for n in need:
            self.table.append([order.pop() for _ in range(n)] + [order[0]] * (width - n))
        rows = torch.randn((2, P, heads, ps, 128), generator=g).to(BF)
        live = torch.zeros((P, ps), dtype=torch.bool)
        for t, row in zip(lens, self.table):
            for p in range(t):
                live[row[p // ps], p % ps] = True
        live = live[:, None, :].expand(P, heads, ps)
        nan = float("nan")
        if dtype == BF:
            self.raw = torch.where(live[None, ..., None], rows, torch.full_like(rows, nan))
            self.scales = [None, None]
            self.val = self.raw.double()
        else:
            codes, scale = O.quant_rows(rows * torch.tensor([1.0, 2.5])[:, None, None, None, None], dtype)
            stored = codes.float().to(torch.float8_e4m3fn).view(torch.uint8) if dtype == E4 else codes.to(S8)
            self.raw = torch.where(live[None, ..., None], stored, torch.full_like(stored, 0x7F))
            s = torch.where(live[None], scale, torch.full_like(scale, nan)).float()
            self.scales = [s[0].to(DEV), s[1].to(DEV)]
            self.val = O.code_values(self.raw) * s.double()[..., None]
        dev = [self.raw[i].to(DEV) for i in range(2)]
        if token_major:  # pages stored [page, row, head, 128], seen through a transposed view
            dev = [d.transpose(1, 2).contiguous().transpose(1, 2) for d in dev]
        self.pages = K().KVPages(dev[0], dev[1], *self.scales)

    def plan(self, new):
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        t = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
        return cu, (t(self.table), t(cu), t(self.lens))


def tolerance(ref, mag, d=0.0):
    extra = 2 ** -11 + math.expm1(2 * d) if d else 0.0
    return (2 ** -8 + 5e-4 + extra) * mag + 2 ** -8 * ref.abs() + 1e-30


def close(out, lse, ref, ref_lse, mag, d=0.0):
    """``d``: the most that a score moves by its key's rounding to f16, 0 for bf16 keys."""
    o, l = out.double().cpu(), lse.double().cpu()
    tol = tolerance(ref, mag, d)
    bad = ~((o - ref).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), float(((o - ref).abs() / tol).nan_to_num(9e9).max()))
    none = torch.isinf(ref_lse)
    assert torch.equal(torch.isinf(l), none)
    err = (l - ref_lse)[~none].abs()
    assert (err <= 2e-4 + d + 1e-6 * ref_lse[~none].abs()).all(), float(err.max())


def check_attention(pool, new, H, block=0, window=0, sink=0, q_scale=1.0, seed=0, hints=(None, None), tail=0, q=None):
    cu, plan = pool.plan(new)
    rows = cu[-1] + tail
    g = torch.Generator().manual_seed(seed + 1)
    if q is None:
        q = (torch.randn((rows, H, 128), generator=g) * q_scale).to(BF)
    out = torch.full((rows, H, 128), 7.0, dtype=BF, device=DEV)
    got, lse = K().paged_attention(q.to(DEV), pool.pages, *plan, max_new=hints[0], max_len=hints[1], block=block,
                                   window=window, sink=sink, out=out, return_lse=True)
    ref, ref_lse, written = O.paged_attention(q[:cu[-1]], *pool.val, pool.table, cu, pool.lens, block, window, sink, SCALE)
    mag, _, _ = O.paged_attention(q[:cu[-1]], pool.val[0], pool.val[1].abs(), pool.table, cu, pool.lens, block, window,
                                  sink, SCALE)
    close(got[:cu[-1]], lse[:cu[-1]], ref, ref_lse, mag, score_move(pool, q))
    assert (got[cu[-1]:] == 7.0).all()  # rows behind the last sequence are left as they were
    return got


CASES = [  # lens, new, H, G, page, block, window, sink
    ([1], [1], 1, 1, 16, 0, 0, 0),
    ([130], [1], 2, 2, 16, 1, 0, 0),
    ([129, 1, 300], [1, 1, 1], 8, 2, 16, 1, 0, 0),
    ([700, 33], [5, 33], 6, 2, 64, 1, 0, 0),
    ([257, 64], [257, 1], 4, 1, 64, 1, 0, 0),
    ([520], [300], 3, 1, 24, 1, 0, 0),
    ([300, 9], [130, 9], 2, 2, 100, 0, 0, 0),
    ([390 * 3], [390], 2, 2, 390, 390, 0, 0),
    ([780], [390], 2, 1, 130, 195, 400, 100),
    ([900], [40], 5, 1, 16, 1, 37, 0),
    ([900], [900], 2, 2, 128, 1, 200, 5),
    ([1000, 0, 40], [64, 0, 40], 4, 4, 128, 0, 0, 0),
    ([600], [1], 4, 2, 48, 1, 100, 20),
    ([2100], [7], 16, 2, 256, 0, 0, 0),
    ([77], [20], 12, 12, 1, 1, 0, 0),
    ([64, 5], [1, 1], 128, 1, 8, 1, 0, 0),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "e4m3", "s8"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"len{c[0]}new{c[1]}h{c[2]}g{c[3]}p{c[4]}b{c[5]}w{c[6]}s{c[7]}")
def test_attention(case, dtype):
    lens, new, H, G, ps, block, window, sink = case
    pool = Pool(dtype, lens, G, ps, seed=len(lens) + H)
    check_attention(pool, new, H, block, window, sink)
    healthy()


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "e4m3", "s8"])
def test_attention_hints_do_not_change_what_is_computed(dtype):
    """max_new / max_len bound the work's split only: exact, loose and wrong ones agree with the oracle."""
    pool = Pool(dtype, [900, 40], 2, 64, seed=3)
    for hints in [(None, None), (30, 900), (1, 16), (5000, 100000)]:
        check_attention(pool, [30, 2], 4, block=1, hints=hints, tail=3)
    healthy()


def test_attention_rows_without_position_or_keys():
    """A sequence shorter than its new rows: the earlier rows see nothing."""
    pool = Pool(BF, [3, 0, 260], 2, 16, seed=4)
    got = check_attention(pool, [5, 2, 200], 2, block=1)
    assert (got[:2] == 0).all() and (got[5:7] == 0).all()
    healthy()


def test_attention_large_logits_and_token_major_pages():
    for dtype in DTYPES:
        pool = Pool(dtype, [1500], 2, 64, seed=5, token_major=True)
        check_attention(pool, [140], 2, block=0, q_scale=20.0)
        check_attention(pool, [3], 4, block=1, q_scale=20.0)
    healthy()


def test_attention_strided_queries():
    pool = Pool(E4, [400], 2, 64, seed=6)
    wide = torch.randn((60, 12, 128), generator=torch.Generator().manual_seed(1)).to(BF)
    q = wide.to(DEV)[:, 4:8]  # heads of a fused projection
    cu, plan = pool.plan([60])
    a = K().paged_attention(q, pool.pages, *plan, block=1)
    b = K().paged_attention(q.contiguous(), pool.pages, *plan, block=1)
    assert torch.equal(a, b)
    healthy()


def test_attention_bad_page_ids_count_as_absent():
    """Ids outside the pool raise the status bit; their keys are absent."""
    from waveforcing_b200 import _lib

    for new, block in (([1], 1), ([150], 0)):
        pool = Pool(BF, [300], 2, 64, seed=7)
        pool.table[0][1], pool.table[0][3] = -5, 10 ** 6
        check_attention(pool, new, 2, block=block)
        assert _lib.status_take() == 1 << 9


def test_attention_replays_with_new_lengths():
    """One captured call serves later steps: page table, offsets and lengths are device data."""
    pool = Pool(E4, [500, 90], 2, 16, seed=8)
    cu, plan = pool.plan([1, 1])
    q = torch.randn((2, 4, 128), device=DEV).to(BF)
    out = torch.zeros_like(q)
    run = lambda: K().paged_attention(q, pool.pages, *plan, max_new=1, max_len=512, block=1, out=out)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for lens in ([500, 90], [17, 3], [129, 64]):
        plan[2].copy_(torch.tensor(lens, dtype=torch.int32))
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(lens[0])))
        graph.replay()
        torch.cuda.synchronize()
        ref, _, _ = O.paged_attention(q.cpu(), *pool.val, pool.table, cu, lens, 1, 0, 0, SCALE)
        mag, _, _ = O.paged_attention(q.cpu(), pool.val[0], pool.val[1].abs(), pool.table, cu, lens, 1, 0, 0, SCALE)
        assert ((out.double().cpu() - ref).abs() <= tolerance(ref, mag, score_move(pool, q.cpu()))).all()
    healthy()


# ------------------------------------------------------------------ the cache
def special_rows(x):
    """Rows of zeros, of tiny and huge values, exact rounding midpoints."""
    x[0] = 0
    x[1] = 2.0 ** -120
    x[2] = torch.linspace(-1, 1, 128) * 3e38
    x[3] = (torch.arange(128) - 63).float()  # with amax 64: midpoints of both codecs
    x[4, :, 0] = 255 * 2.0 ** 60
    return x


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "e4m3", "s8"])
@pytest.mark.parametrize("lens,new,G,ps", [([40], [40], 3, 16), ([1], [1], 1, 1560), ([130, 7, 64], [50, 1, 64], 5, 24),
                                           ([3, 2000], [2, 90], 12, 64)])
def test_write_and_read_back(dtype, lens, new, G, ps):
    pool = Pool(dtype, lens, G, ps, seed=9)
    cu, plan = pool.plan(new)
    rows, tail = cu[-1], 2
    g = torch.Generator().manual_seed(10)
    k = (torch.randn((rows + tail, G, 128), generator=g) * 3).to(BF)
    v = torch.randn((rows + tail, G, 128), generator=g).to(BF)
    if rows > 8:
        k[:8] = special_rows(k[:8].float()).to(BF)
    before = [t.clone() for t in (pool.pages.k, pool.pages.v)]
    K().paged_kv_write(pool.pages, k.to(DEV), v.to(DEV), *plan)
    touched = torch.zeros((pool.P, ps), dtype=torch.bool)
    for i, x in enumerate((k, v)):
        stored = (pool.pages.k, pool.pages.v)[i].cpu()
        codes, scale = O.quant_rows(x, dtype) if dtype != BF else (x.double(), None)
        for r, _, page, row in O.slots(pool.table, cu, lens, ps, pool.P):
            touched[page, row] = True
            assert torch.equal(O.code_values(stored)[page, :, row], codes[r]), (i, r)
            if scale is not None:
                got = pool.scales[i].cpu()[page, :, row].double()
                assert ((got - scale[r]).abs() <= 2 ** -24 * scale[r]).all()
        keep = ~touched[:, None, :, None].expand_as(stored)
        assert torch.equal(stored.view(torch.uint8)[keep.repeat_interleave(stored.element_size(), -1)],
                           before[i].cpu().view(torch.uint8)[keep.repeat_interleave(stored.element_size(), -1)])
    out = [torch.full((rows + tail, G, 128), 7.0, dtype=BF, device=DEV) for _ in range(2)]
    K().paged_kv_read(pool.pages, *plan, out_k=out[0], out_v=out[1])
    for i, x in enumerate((k, v)):
        assert (out[i][rows:] == 7.0).all()
        want = x[:rows].double()
        if dtype != BF:
            codes, scale = O.quant_rows(x[:rows], dtype)
            want = codes * scale[..., None]
        assert ((out[i][:rows].double().cpu() - want).abs() <= (2 ** -8 + 2 ** -23) * want.abs()).all()
    healthy()


@pytest.mark.parametrize("dtype", [E4, S8], ids=["e4m3", "s8"])
def test_rows_that_are_not_finite_read_back_as_nan(dtype):
    pool = Pool(dtype, [20], 2, 16, seed=11)
    cu, plan = pool.plan([4])
    k = torch.randn((4, 2, 128)).to(BF)
    k[1, 0, 5], k[2, 1, 0], k[3, 0, 127] = float("nan"), float("inf"), -float("inf")
    v = torch.randn((4, 2, 128)).to(BF)
    K().paged_kv_write(pool.pages, k.to(DEV), v.to(DEV), *plan)
    rk, rv = K().paged_kv_read(pool.pages, *plan, rows=4)
    bad = torch.zeros((4, 2), dtype=torch.bool)
    bad[1, 0] = bad[2, 1] = bad[3, 0] = True
    assert torch.equal(torch.isnan(rk).all(-1).cpu(), bad) and torch.equal(torch.isnan(rk).any(-1).cpu(), bad)
    assert torch.isfinite(rv).all()
    q = torch.randn((4, 2, 128)).to(BF).to(DEV)
    o = K().paged_attention(q, pool.pages, *plan, block=1)
    # row 0 sees none of the bad keys; head 0 is lost from row 1 on, head 1 from row 2 on
    want = torch.tensor([[False, False], [True, False], [True, True], [True, True]])
    assert torch.equal(torch.isnan(o).any(-1).cpu(), want)
    healthy()


def test_write_into_a_page_listed_twice_keeps_the_later_row():
    for dtype in DTYPES:
        pages = K().KVPages.empty(4, 3, 16, dtype, DEV)
        t = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
        k = torch.randn((56, 3, 128)).to(BF).to(DEV)
        # two sequences whose newest rows share page 2, and one that lists page 1 twice
        table, cu, lens = t([[0, 2], [3, 2], [1, 1]]), t([0, 12, 24, 56]), t([28, 28, 32])
        for _ in range(5):
            K().paged_kv_write(pages, k, k, table, cu, lens)
            rk, _ = K().paged_kv_read(pages, table, cu, lens, rows=56)
            one = K().KVPages.empty(4, 3, 16, dtype, DEV)
            K().paged_kv_write(one, k[12:24], k[12:24], t([[3, 2]]), t([0, 12]), t([28]))
            K().paged_kv_write(one, k[40:], k[40:], t([[1]]), t([0, 16]), t([16]))
            wk, _ = K().paged_kv_read(one, t([[3, 2], [1, 1]]), t([0, 12, 44]), t([28, 32]), rows=44)
            assert torch.equal(rk[:12], wk[:12]) and torch.equal(rk[12:24], wk[:12]) and torch.equal(rk[24:], wk[12:])
    healthy()


def test_write_and_read_of_bad_pages():
    from waveforcing_b200 import _lib

    pool = Pool(E4, [40], 2, 16, seed=12)
    pool.table[0][1] = pool.P + 3
    cu, plan = pool.plan([40])
    k = torch.randn((40, 2, 128)).to(BF).to(DEV)
    K().paged_kv_write(pool.pages, k, k, *plan)
    rk, _ = K().paged_kv_read(pool.pages, *plan, rows=40)
    assert _lib.status_take() == 1 << 9
    assert (rk[16:32] == 0).all() and torch.isfinite(rk).all() and (rk[:16] != 0).any()


# ------------------------------------------------------------ cross attention
CROSS = [  # B, Lq, N, Lk, H, G, lens, mask, index
    (1, 1, 1, 1, 1, 1, None, False, None),
    (2, 300, 2, 77, 2, 2, None, False, None),
    (3, 130, 3, 512, 4, 4, [512, 20, 0], False, None),
    (4, 1, 4, 257, 8, 2, None, True, None),
    (3, 40, 1, 100, 6, 1, [63], True, None),
    (5, 70, 2, 200, 2, 2, [200, 130], True, [1, 0, 0, 1, 1]),
    (1, 600, 1, 1030, 3, 3, None, True, None),
    (2, 5, 2, 3, 40, 40, [3, 1], False, None),
]


@pytest.mark.parametrize("case", CROSS, ids=lambda c: f"B{c[0]}q{c[1]}n{c[2]}k{c[3]}h{c[4]}g{c[5]}m{int(c[7])}")
def test_cross_attention(case):
    B, Lq, N, Lk, H, G, lens, masked, index = case
    g = torch.Generator().manual_seed(B * 100 + Lq)
    q = torch.randn((B, Lq, H, 128), generator=g).to(BF)
    k, v = (torch.randn((N, Lk, G, 128), generator=g).to(BF) for _ in range(2))
    mask = torch.rand((N, Lk), generator=g) < 0.6 if masked else None
    if masked and N > 1:
        mask[1] = False  # a state set that keeps nothing
    seen = torch.ones((N, Lk), dtype=torch.bool) if mask is None else mask.clone()
    if lens is not None:
        seen &= torch.arange(Lk) < torch.tensor(lens)[:, None]
    k[~seen], v[~seen] = float("nan"), float("inf")  # what is masked does not matter
    t = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    out, lse = K().cross_attention(q.to(DEV), k.to(DEV), v.to(DEV), kv_lens=t(lens),
                                   key_mask=None if mask is None else mask.to(DEV), kv_index=t(index), return_lse=True)
    ref, ref_lse = O.cross_attention(q, k, v, lens, mask, index, SCALE)
    mag, _ = O.cross_attention(q, k, v.abs(), lens, mask, index, SCALE)
    close(out, lse, ref, ref_lse, mag)
    healthy()


def test_cross_attention_bad_index():
    from waveforcing_b200 import _lib

    q = torch.randn((3, 9, 2, 128), device=DEV).to(BF)
    k = torch.randn((2, 50, 2, 128), device=DEV).to(BF)
    out = K().cross_attention(q, k, k, kv_index=torch.tensor([0, 2, -1], dtype=torch.int32, device=DEV))
    assert _lib.status_take() == 1 << 9
    assert (out[1:] == 0).all() and (out[0] != 0).any()


def test_write_then_attend_then_cross_as_a_layer_does():
    """A run of them together: two steps of two sequences through write,
    attention over the pages and cross attention, against the f64 oracle on what
    the cache stands for."""
    torch.manual_seed(0)
    H, G, ps = 4, 2, 16
    pages = K().KVPages.empty(12, G, ps, E4, DEV)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    table = [[3, 7, 1, 9], [2, 5, 11, 0]]
    text, tl = torch.randn((2, 30, G, 128)).to(BF), [30, 11]
    hist = [[], []]
    lens = [0, 0]
    for new in ([33, 20], [1, 1], [1, 1]):
        lens = [a + n for a, n in zip(lens, new)]
        cu = [0, new[0], sum(new)]
        k, v, q = (torch.randn((sum(new), h, 128)).to(BF) for h in (G, G, H))
        plan = (t(table), t(cu), t(lens))
        K().paged_kv_write(pages, k.to(DEV), v.to(DEV), *plan)
        o = K().paged_attention(q.to(DEV), pages, *plan, block=1)
        for b in range(2):
            hist[b].append([O.quant_rows(x[cu[b]:cu[b + 1]], E4) for x in (k, v)])
            kk, vv = (torch.cat([h[i][0] * h[i][1].float().double()[..., None] for h in hist[b]]) for i in range(2))
            keep = torch.stack([O.visible(lens[b] - new[b] + i, lens[b], 1, 0, 0) for i in range(new[b])])
            for h in range(H):
                args = (q[cu[b]:cu[b + 1], h], kk[:, h // 2])
                ref, _ = O.softmax_rows(*args, vv[:, h // 2], keep, SCALE)
                mag, _ = O.softmax_rows(*args, vv[:, h // 2].abs(), keep, SCALE)
                err = (o[cu[b]:cu[b + 1], h].double().cpu() - ref).abs()
                assert (err <= tolerance(ref, mag, most_move(*args))).all()
        if new[0] == new[1]:
            x = o.view(2, 1, H, 128)
            c = K().cross_attention(x, text.to(DEV), text.to(DEV), kv_lens=t(tl))
            ref, _ = O.cross_attention(x.cpu(), text, text, tl, None, None, SCALE)
            mag, _ = O.cross_attention(x.cpu(), text, text.abs(), tl, None, None, SCALE)
            assert ((c.double().cpu() - ref).abs() <= tolerance(ref, mag)).all()
    healthy()


def test_calls_on_another_stream_and_two_at_once():
    """Two calls in flight on two streams keep to their own workspaces."""
    pool = Pool(E4, [3000, 900], 2, 64, seed=13)
    cu, plan = pool.plan([1, 1])
    q = [torch.randn((2, 8, 128), device=DEV).to(BF) for _ in range(2)]
    want = [K().paged_attention(x, pool.pages, *plan, max_new=1, block=1) for x in q]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        got = []
        for s, x in zip(streams, q):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(K().paged_attention(x, pool.pages, *plan, max_new=1, block=1))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    healthy()


def test_log_sum_exp_joins_two_halves_of_a_context():
    """return_lse lets a caller join attention over two parts of a context."""
    pool = Pool(BF, [512], 2, 64, seed=14)
    cu, plan = pool.plan([4])
    q = torch.randn((4, 2, 128), device=DEV).to(BF)
    whole, lse = K().paged_attention(q, pool.pages, *plan, return_lse=True)
    parts = []
    for ids in (pool.table[0][:4], pool.table[0][4:]):
        tb = torch.tensor([ids], dtype=torch.int32, device=DEV)
        parts.append(K().paged_attention(q, pool.pages, tb, plan[1], torch.tensor([256], dtype=torch.int32, device=DEV),
                                         return_lse=True))
    m = torch.logaddexp(parts[0][1], parts[1][1])
    o = sum(p[0].float() * torch.exp(p[1] - m)[..., None] for p in parts)
    # 2e-4 for each side's lse, whose difference the weights carry over; on each side the header's bound, with |o| <= A
    assert (m - lse).abs().max() <= 4e-4
    mag, _, _ = O.paged_attention(q.cpu(), pool.val[0], pool.val[1].abs(), pool.table, cu, pool.lens, 0, 0, 0, SCALE)
    assert ((o - whole.float()).abs().double().cpu() <= (4 * 2 ** -8 + 2 * 5e-4 + 4e-4) * mag).all()
    healthy()


LONG = [  # lens, new, H, G, page, block: one sequence's items dealt out in parts, or several sequences' keys split
    ([2500], [300], 12, 12, 64, 1),      # 24 items: all in parts
    ([2200], [600], 50, 50, 128, 0),     # 150 items: a round of whole ones, two in parts
    ([3301], [200], 4, 2, 48, 100),      # pages that do not divide a tile
    ([5000, 3000], [20, 17], 4, 2, 16, 1),
    ([4100, 1, 2050], [40, 1, 3], 2, 2, 128, 0),
    ([3300], [260], 2, 1, 1560, 390),    # tiles across the ends of large pages
    ([1700], [150], 3, 3, 200, 50),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "e4m3", "s8"])
@pytest.mark.parametrize("case", LONG, ids=lambda c: f"len{c[0]}new{c[1]}h{c[2]}p{c[4]}")
def test_attention_in_parts(case, dtype):
    lens, new, H, G, ps, block = case
    pool = Pool(dtype, lens, G, ps, seed=len(lens) + H)
    check_attention(pool, new, H, block, hints=(max(new), max(lens)))
    check_attention(pool, new, H, block, window=700, sink=130, tail=1)
    healthy()


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "e4m3", "s8"])
@pytest.mark.parametrize("block,window,sink", [(1, 0, 0), (64, 500, 40)])
def test_attention_of_ragged_prompts(dtype, block, window, sink):
    """More items than run at once, taken from the longest to the shortest; one sequence has no new
    rows, one is shorter than its new rows, and rows lie behind the last."""
    pool = Pool(dtype, [1500, 40, 300, 7, 900, 2000], 6, 16, seed=17)
    check_attention(pool, [700, 40, 0, 9, 300, 900], 24, block, window, sink, hints=(900, 2000), tail=3)
    healthy()


@pytest.mark.parametrize("dtype", [E4, S8], ids=["e4m3", "s8"])
def test_scales_with_strides_of_their_own(dtype):
    pool = Pool(dtype, [400, 90], 2, 64, seed=15)
    cu, plan = pool.plan([150, 1])
    p = pool.pages
    wide = [torch.full((pool.P, 3, 67), float("nan"), device=DEV) for _ in range(2)]
    for w, s in zip(wide, (p.k_scale, p.v_scale)):
        w[:, :2, 1:65] = s
    odd = K().KVPages(p.k, p.v, wide[0][:, :2, 1:65], wide[1][:, :2, 1:65])
    for rows, block in ((151, 0), (151, 1)):
        q = torch.randn((rows, 4, 128), device=DEV).to(BF)
        assert torch.equal(K().paged_attention(q, p, *plan, block=block), K().paged_attention(q, odd, *plan, block=block))
    cu1, plan1 = pool.plan([1, 1])
    q = torch.randn((2, 4, 128), device=DEV).to(BF)
    assert torch.equal(K().paged_attention(q, p, *plan1, max_new=1), K().paged_attention(q, odd, *plan1, max_new=1))
    k = torch.randn((151, 2, 128), device=DEV).to(BF)
    for pages in (p, odd):
        K().paged_kv_write(pages, k, k, *plan)
    for a, b in zip(K().paged_kv_read(p, *plan, rows=151), K().paged_kv_read(odd, *plan, rows=151)):
        assert torch.equal(a, b)
    # what lies beside the scales is left alone
    assert wide[0][:, 2].isnan().all() and wide[0][:, :, 0].isnan().all() and wide[0][:, :, 65:].isnan().all()
    healthy()


@pytest.mark.parametrize("dtype", [BF, E4], ids=["bf16", "e4m3"])
def test_pools_of_more_than_2_to_the_31_elements(dtype):
    """Page offsets in 64 bits: the same rows through the first and the last pages of a large pool."""
    ps, G = 64, 2
    P = 2 ** 31 // (ps * G * 128) + 40
    kv = [torch.empty((P, G, ps, 128), dtype=dtype, device=DEV) for _ in range(2)]
    pages = K().KVPages(*kv, *([] if dtype == BF else [torch.empty((P, G, ps), device=DEV) for _ in range(2)]))
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    cu, lens = t([0, 300]), t([300])
    k, v = (torch.randn((300, G, 128), device=DEV).to(BF) for _ in range(2))
    q = torch.randn((300, 4, 128), device=DEV).to(BF)
    got = []
    for table in ([[0, 1, 2, 3, 4]], [[P - 1, P - 3, P - 5, 2, P - 2]]):
        K().paged_kv_write(pages, k, v, t(table), cu, lens)
        got.append([*K().paged_kv_read(pages, t(table), cu, lens, rows=300),
                    K().paged_attention(q, pages, t(table), cu, lens, block=1),
                    K().paged_attention(q[-2:], pages, t(table), t([0, 2]), lens, block=1)])
    for a, b in zip(*got):
        assert torch.isfinite(a).all() and torch.equal(a, b)
    healthy()


def test_two_graphs_replayed_at_once_keep_their_workspaces():
    pool = Pool(BF, [4000, 2500], 2, 64, seed=16)
    cu, plan = pool.plan([1, 1])
    q = [torch.randn((2, 2, 128), device=DEV).to(BF) for _ in range(2)]
    q += [torch.randn((40, 2, 128), device=DEV).to(BF) for _ in range(2)]
    long = pool.plan([20, 20])[1]
    call = lambda x: K().paged_attention(x, pool.pages, *(plan if len(x) == 2 else long),  # noqa: E731
                                         max_new=len(x) // 2, max_len=4000, block=1)
    want = [call(x) for x in q]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in q:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(call(x))
    streams = [torch.cuda.Stream() for _ in q]
    for _ in range(10):
        for o in outs:
            o.zero_()
        for s, g in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    healthy()


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "e4m3", "s8"])
def test_write_and_read_of_many_heads(dtype):
    """Enough rows that a block walks several groups of heads, the last of them not full."""
    rows, G, ps = 4800, 37, 64
    pages = K().KVPages.empty(rows // ps + 1, G, ps, dtype, DEV)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    plan = (t([list(range(rows // ps, -1, -1))]), t([0, rows]), t([rows + 5]))
    x = [torch.randn((rows, G, 128), generator=torch.Generator().manual_seed(i)).to(BF) for i in range(2)]
    K().paged_kv_write(pages, x[0].to(DEV), x[1].to(DEV), *plan)
    for a, b in zip(K().paged_kv_read(pages, *plan, rows=rows), x):
        if dtype == BF:
            assert torch.equal(a.cpu(), b)
            continue
        codes, scale = O.quant_rows(b, dtype)
        want = codes * scale[..., None]
        assert ((a.double().cpu() - want).abs() <= (2 ** -8 + 2 ** -23) * want.abs()).all()
    healthy()


def test_cross_attention_into_rows_that_are_not_32_byte_aligned():
    """Outputs whose rows start on 16-byte boundaries only."""
    q = torch.randn((2, 200, 3, 128), device=DEV).to(BF)
    k = torch.randn((2, 300, 3, 128), device=DEV).to(BF)
    want = K().cross_attention(q, k, k)
    room = torch.full((2, 200, 3, 136), 7.0, device=DEV, dtype=BF)
    K().cross_attention(q, k, k, out=room[..., 8:])
    assert torch.equal(room[..., 8:], want) and (room[..., :8] == 7.0).all()
    healthy()


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "e4m3", "s8"])
def test_single_tokens_of_many_sequences(dtype):
    """Each CTA of the few-row kernel walks several sequences, over runs of such as have no new token."""
    g = torch.Generator().manual_seed(21)
    lens = torch.randint(0, 200, (700,), generator=g).tolist()
    new = (torch.rand(700, generator=g) < 0.7).int().tolist()
    new[100:150] = [0] * 50
    pool = Pool(dtype, lens, 2, 16, seed=22)
    check_attention(pool, new, 4, block=1, hints=(1, 200))
    lens = torch.randint(1, 3000, (40,), generator=g).tolist()  # cut into equal stretches
    new = (torch.rand(40, generator=g) < 0.7).int().tolist()
    pool = Pool(dtype, lens, 2, 64, seed=23)
    check_attention(pool, new, 4, block=1, hints=(1, 3000))
    healthy()


def set_keys(pool, rows):
    """Gives the first len(rows) positions of the only sequence (all heads) the K rows `rows` [n, 128] f64,
    quantised as the write does; rows of zeros by turns as written (scale 2^-100 / Q) and as never written."""
    for p, x in enumerate(rows):
        page, row = pool.table[0][p // pool.ps], p % pool.ps
        if pool.dtype == BF:
            pool.pages.k[page, :, row] = x.to(BF).to(DEV)
            pool.val[0][page, :, row] = x.to(BF).double()
            continue
        codes, scale = O.quant_rows(x.to(BF), pool.dtype)
        scale = scale.float() * (0.0 if p % 2 and not x.any() else 1.0)
        stored = codes.float().to(torch.float8_e4m3fn).view(torch.uint8) if pool.dtype == E4 else codes.to(S8)
        pool.pages.k[page, :, row], pool.pages.k_scale[page, :, row] = stored.to(DEV), scale.to(DEV)
        pool.val[0][page, :, row] = codes * scale.double()


# new tokens: the few-row and the many-row kernel, one and two sub-tiles
NEW = [3, 100, 150]


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "e4m3", "s8"])
@pytest.mark.parametrize("new", NEW)
@pytest.mark.parametrize("block", [0, 1])
def test_queries_and_keys_of_zeros(dtype, new, block):
    """Scores of 0 in tiles that end inside and that rows see in part: the mean of V, not NaN."""
    for tiny in (0.0, 2.0 ** -120):
        q = torch.full((new, 2, 128), tiny).to(BF)
        q[::3] = torch.randn((len(q[::3]), 2, 128), generator=torch.Generator().manual_seed(30)).to(BF)
        pool = Pool(dtype, [300], 2, 64, seed=31)
        check_attention(pool, [new], 2, block, q=q)  # zero queries over ordinary keys
        check_attention(pool, [new], 2, block, window=130, sink=3, q=q)
        set_keys(pool, torch.zeros(300, 128, dtype=torch.float64))
        check_attention(pool, [new], 2, block, q=q)
        check_attention(pool, [new], 2, block, window=130, sink=3, q=q)
    healthy()


@pytest.mark.parametrize("dtype", [E4, S8], ids=["e4m3", "s8"])
def test_an_empty_pool_gives_zeros(dtype):
    """As a warm-up calls it: zero queries over pages that were never written."""
    pages = K().KVPages.empty(8, 2, 64, dtype, DEV)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    for new in NEW:
        q = torch.zeros((new, 4, 128), dtype=BF, device=DEV)
        o, lse = K().paged_attention(q, pages, t([list(range(8))]), t([0, new]), t([300]), return_lse=True)
        assert (o == 0).all() and (lse - math.log(300)).abs().max() <= 2e-4 + 1e-6 * math.log(300)
    healthy()


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "e4m3", "s8"])
@pytest.mark.parametrize("ps", [16, 48, 128])
def test_bad_page_ids_over_every_type(dtype, ps):
    """Whole tiles and parts of them out of the pool; zero query rows among the others."""
    from waveforcing_b200 import _lib

    for new in NEW:
        pool = Pool(dtype, [700], 2, ps, seed=32)
        for j in [0, 1, *range(256 // ps, 384 // ps), -1]:
            pool.table[0][j] = -5 if j % 2 else 10 ** 6
        q = torch.randn((new, 4, 128), generator=torch.Generator().manual_seed(33)).to(BF)
        q[::2] = 0
        for block in (0, 1):
            check_attention(pool, [new], 4, block, q=q)
            assert _lib.status_take() == 1 << 9


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "e4m3", "s8"])
@pytest.mark.parametrize("new", NEW)
def test_products_beyond_f32(dtype, new):
    """|q| |k| above f32's range where q.k is 0 (a score of 0) or far below 0 (no weight)."""
    keys = torch.randn((300, 128), generator=torch.Generator().manual_seed(34)).double()
    keys[:, :2] = 0
    keys[5], keys[200] = 0.0, 0.0
    keys[5, 1], keys[200, 0] = 2.0 ** 100, -(2.0 ** 100)
    q = torch.zeros((new, 2, 128))
    q[..., 0] = 2.0 ** 100
    pool = Pool(dtype, [300], 2, 64, seed=35)
    set_keys(pool, keys)
    cu, plan = pool.plan([new])
    got, lse = K().paged_attention(q.to(BF).to(DEV), pool.pages, *plan, return_lse=True)
    ref, ref_lse, _ = O.paged_attention(q.to(BF), *pool.val, pool.table, cu, pool.lens, 0, 0, 0, SCALE)
    mag, _, _ = O.paged_attention(q.to(BF), pool.val[0], pool.val[1].abs(), pool.table, cu, pool.lens, 0, 0, 0, SCALE)
    close(got, lse, ref, ref_lse, mag, 0.0 if dtype == BF else 2 ** -11)  # every score is 0 or has no weight: none moves
    healthy()


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "e4m3", "s8"])
def test_scores_beyond_2_to_the_28(dtype):
    """Few rows with scores of about 2^34, where f32 has steps of 2^10: the largest takes all."""
    g = torch.Generator().manual_seed(36)
    keys = (torch.randn((300, 128), generator=g) * 2.0 ** 16).double()
    q = (torch.randn((3, 2, 128), generator=g) * 2.0 ** 18).to(BF)
    pool = Pool(dtype, [300], 2, 64, seed=37)
    set_keys(pool, keys)
    cu, plan = pool.plan([3])
    got = K().paged_attention(q.to(DEV), pool.pages, *plan).double().cpu()
    k, v = (torch.cat([pool.val[i][page] for page in pool.table[0]], 1)[:, :300] for i in range(2))  # [heads, keys, 128]
    s = torch.einsum("rhd,hkd->rhk", q.double(), k) * SCALE
    top = s.topk(2, -1)
    assert (top.values[..., 0] - top.values[..., 1]).min() > 2.0 ** 20  # far above f32's steps of the sum
    want = torch.stack([v[h][top.indices[:, h, 0]] for h in range(2)], 1)
    assert ((got - want).abs() <= (2 ** -8 + (0 if dtype == BF else 2 ** -11)) * want.abs()).all()
    healthy()


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "e4m3", "s8"])
@pytest.mark.parametrize("new,H,G,L,sink_at", [
    (3, 1, 1, 4200, 0), (3, 1, 1, 4200, 2050), (3, 1, 1, 4200, 4199), (3, 1, 1, 32768, 0),  # few rows
    (150, 1, 1, 4200, 0), (150, 1, 1, 32768, 0),                                            # in parts
    (400, 128, 2, 1900, 0), (400, 128, 2, 1900, 1030), (400, 128, 2, 1900, 1899)])          # whole items
@pytest.mark.parametrize("sink", ["empty", "tiny", "like"])
def test_weights_far_below_the_largest(dtype, new, H, G, L, sink_at, sink):
    """One key takes nearly all weight, as an attention sink does, and has no V, little or as much as the
    others, whose weights are e^-8 to e^-16 of its own.

    The scores are exact (one product of powers of two, or 0) so that d is 0.  Over 8-bit pages weights
    are f16 with the largest at least 2^7 (many rows) or 2^13 times V's scale over a power of two that is at
    most 4 times the largest scale (few rows): half of f16's smallest step is 2^-25, so each key may lose
    2^-25 / 2^7 of the largest weight times its |v|, or 2^-25 / 2^13 * 4 times the largest |v|."""
    g = torch.Generator().manual_seed(40)
    k = torch.zeros((L, G, 128))
    k[sink_at, :, 0] = 16.0
    v = torch.randn((L, G, 128), generator=g) + 0.5
    if sink == "like":
        v[:] = v[1]
    else:
        v[sink_at] = 0.0 if sink == "empty" else 2.0 ** -20
    k, v = k.to(BF), v.to(BF)
    q = torch.zeros((4, 128))
    q[:, 0] = torch.tensor([12.0, 14.0, 16.0, 8.0]) / (16 * SCALE)
    q = q.to(BF)
    kind = torch.arange(new) % 4
    ps = 64
    pages = K().KVPages.empty(L // ps + 1, G, ps, dtype, DEV)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    table = t([list(range(L // ps, -1, -1))])
    K().paged_kv_write(pages, k.to(DEV), v.to(DEV), table, t([0, L]), t([L]))
    o, lse = K().paged_attention(q[kind][:, None].expand(new, H, 128).contiguous().to(DEV), pages, table, t([0, new]), t([L]),
                                 return_lse=True)
    o, lse = o.double().cpu().view(new, G, H // G, 128), lse.double().cpu().view(new, G, H // G)
    if dtype == BF:
        kk, vv, lost = k.double(), v.double(), 0.0
    else:
        kk, vv = ((c * s.float().double()[..., None]) for c, s in (O.quant_rows(x, dtype) for x in (k, v)))
        lost = 2 ** -38 * 4 if new == 3 else 2 ** -32
    keep = torch.ones((4, L), dtype=torch.bool)
    for h in range(G):
        ref, ref_lse = O.softmax_rows(q, kk[:, h], vv[:, h], keep, SCALE)
        mag, _ = O.softmax_rows(q, kk[:, h], vv[:, h].abs(), keep, SCALE)
        # (the sum of weights over the largest is at least 1; of A this is 2e-3 at most, at e^-16)
        small = L * lost * (float(vv.abs().max()) if new == 3 else vv[:, h].abs().mean(0))
        tol = (2 ** -8 + 5e-4 + (2 ** -11 if dtype != BF else 0.0)) * mag + 2 ** -8 * ref.abs() + small
        err = (o[:, h] - ref[kind][:, None]).abs() / tol[kind][:, None]
        assert (err <= 1).all(), float(err.max())
        assert ((lse[:, h] - ref_lse[kind][:, None]).abs() <= 2e-4 + 1e-6 * ref_lse.abs().max()).all()
    healthy()


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "e4m3", "s8"])
def test_what_an_earlier_call_left_on_the_chip_does_not_matter(dtype):
    """Groups that do not divide 128 leave rows of a Q tile without a token."""
    pool = Pool(dtype, [2500], 4, 64, seed=50)
    nan = torch.full((1200, 4, 128), float("nan"), dtype=BF, device=DEV)
    for H in (12, 20, 24):
        K().paged_attention(nan, pool.pages, *pool.plan([1200])[1])
        check_attention(pool, [130], H, block=1)
    healthy()


@pytest.mark.parametrize("lens,new,ps,block,window,sink", [
    ([300], [3], 64, 1, 0, 0), ([300, 40], [7, 7], 16, 1, 50, 3), ([130], [8], 24, 1, 20, 5),    # few rows
    ([300], [100], 64, 1, 0, 0), ([300, 90], [150, 70], 48, 1, 0, 0), ([500], [260], 16, 1, 60, 5),
    ([900], [300], 100, 64, 200, 90), ([2500], [300], 390, 195, 0, 0), ([2500], [200], 128, 1, 700, 130)])
def test_values_that_are_not_finite_reach_only_rows_that_see_them(lens, new, ps, block, window, sink):
    """bf16 pages, where single elements of V may be NaN or infinite: each reaches its own dim of the rows
    that see its key, and no other."""
    pool = Pool(BF, lens, 2, ps, seed=60)
    cu, plan = pool.plan(new)
    g = torch.Generator().manual_seed(61)
    q = torch.randn((cu[-1], 4, 128), generator=g).to(BF)
    odd = torch.zeros_like(pool.val[1])  # what is not finite, by slot
    for b, n in enumerate(lens):
        at = [n - 1, n - 2, n - new[b] // 2, n - new[b], max(n - new[b] - 1, 0), 0, 4, max(n - window - 2, 0), n - n // 3]
        for i, p in enumerate(at):
            page, row, head = pool.table[b][p // ps], p % ps, i % 2
            bad = [float("nan"), float("inf"), -float("inf")][i % 3]
            dims = slice(0, 128) if i == 3 else torch.randint(0, 128, (3,), generator=g)
            odd[page, head, row, dims] = bad
    is_odd = odd != 0
    pool.pages.v[is_odd.to(DEV)] = odd[is_odd].to(BF).to(DEV)
    pool.val[1][is_odd] = 0.0  # the oracle sums what is finite
    got = K().paged_attention(q.to(DEV), pool.pages, *plan, block=block, window=window, sink=sink)
    args = (pool.table, cu, pool.lens, block, window, sink, SCALE)
    ref, _, _ = O.paged_attention(q, *pool.val, *args)
    mag, _, _ = O.paged_attention(q, pool.val[0], pool.val[1].abs(), *args)
    for b, n in enumerate(lens):
        v = torch.cat([odd[page] for page in pool.table[b]], 1)[:, :n]  # [heads, keys, 128]
        for i in range(new[b]):
            keep = O.visible(n - new[b] + i, n, block, window, sink)
            for h in range(4):
                ref[cu[b] + i, h] += v[h // 2][keep].sum(0)
    o, fin = got.double().cpu(), torch.isfinite(ref)
    assert 0 < (~fin).sum() < fin.numel()
    assert torch.equal(torch.isfinite(o), fin)
    assert torch.equal(torch.isnan(o), torch.isnan(ref)) and torch.equal(o[torch.isinf(ref)], ref[torch.isinf(ref)])
    assert ((o - ref).abs()[fin] <= tolerance(ref, mag)[fin]).all()
    healthy()


@pytest.mark.parametrize("dtype", [BF, E4], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("new", NEW)
def test_maxima_that_pass_2_to_the_16(dtype, new):
    """Scores that grow from 65526 to 65543 (times ln 2) along the keys, where the power that f16 weights
    take for range is given up.  Products of powers of two with the keys' scales, so that no score moves by
    rounding to f16; f32 steps there are 2^-7, and half of one is lost in the product with the scale and
    half in the sum: d = 2^-7 ln 2."""
    q = torch.zeros((new, 2, 128))
    q[..., 0], q[..., 1], q[..., 2] = 32000.0, 116.0, 15.6875
    q[1::3, :, 0] *= -1  # and falls from -65526
    q[2::3, :, 1:] = 0  # all the same
    keys = torch.zeros((1500, 128), dtype=torch.float64)
    keys[:, :2] = 16.0
    keys[:, 2] = torch.tensor([1.0, 2.0, 4.0, 8.0]).repeat_interleave(375)
    pool = Pool(dtype, [1500], 2, 64, seed=70)
    set_keys(pool, keys)
    # (the scale 16 / 448 is rounded to f32, which moves all scores of a row alike, by 2^-24 of them: that is in lse's 1e-6)
    assert torch.allclose(pool.val[0][pool.table[0][0], 0, 0, :3], torch.tensor([16.0, 16.0, 1.0]).double(), rtol=2 ** -24, atol=0)
    cu, plan = pool.plan([new])
    q = q.to(BF)
    for block in (0, 1):
        got, lse = K().paged_attention(q.to(DEV), pool.pages, *plan, block=block, return_lse=True)
        args = (pool.table, cu, pool.lens, block, 0, 0, SCALE)
        ref, ref_lse, _ = O.paged_attention(q, *pool.val, *args)
        mag, _, _ = O.paged_attention(q, pool.val[0], pool.val[1].abs(), *args)
        close(got, lse, ref, ref_lse, mag, 2 ** -7 * math.log(2))
    healthy()
