"""The paged key / value cache (ops.kv_cache_write / kv_cache_read), attention of new tokens over it (ops.attn_paged) and the
verification of drafted tokens (ops.draft_verify), against float64.

Tolerances: an e4m3 code is the value nearest to x / scale, so a row reads back within 2^-4 of each element or half the
smallest step (2^-10 scale), plus the rounding of the result; attention as in test_packed.py (worst cases computed beside the
reference), with 64 u more for the products with the scales and the joining of splits.  Verification is whole numbers: equal.
"""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from test_packed import E16, U, reference, within

DEV = "cuda"
E4M3, BF16 = torch.float8_e4m3fn, torch.bfloat16


def _ops():
    from imagecaption_amd import ops
    return ops


def _cast8(x):
    """Float64 values -> nearest e4m3 values (ties to even), written out."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


# ---- write / read -----------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("rows_dtype", [BF16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("dtype", [E4M3, BF16], ids=["cache8", "cache16"])
@pytest.mark.parametrize("rows,heads,page,dh", [(1, 1, 8, 64), (37, 3, 16, 128), (130, 8, 64, 64), (515, 2, 256, 128)])
def test_rows_written_and_read_back(rows, heads, page, dh, dtype, rows_dtype):
    ops = _ops()
    g = torch.Generator().manual_seed(rows)
    pages = -(-rows // page) + 2
    cache = ops.PagedKVCache.new(pages, heads, page, dh, dtype, DEV)
    for t in (cache.k, cache.v):
        t.view(torch.uint8).fill_(0x11)
    for t in (cache.k_scale, cache.v_scale):
        if t is not None:
            t.fill_(7.0)
    wide = torch.randn(rows + 1, 2 * heads * dh + 24, generator=g).mul_(torch.logspace(-6, 4, rows + 1)[:, None]).to(rows_dtype)
    k, v = wide[:rows, 8:8 + heads * dh].to(DEV), wide.to(DEV)[:rows, 16 + heads * dh:16 + 2 * heads * dh]
    slots = torch.randperm(pages * page, generator=g)[:rows].to(torch.int32)
    skipped = torch.zeros(rows, dtype=torch.bool)
    skipped[1::5] = True
    given = torch.where(skipped, -1 - slots, slots)
    before = [t.clone() if t is not None else None for t in (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale)]
    ops.kv_cache_write(cache, k, v, given.to(DEV))
    back = ops.kv_cache_read(cache, given.to(DEV), dtype=torch.float32)
    back16 = ops.kv_cache_read(cache, given.to(DEV))
    page_of, at = slots.long() // page, slots.long() % page
    for x, got, got16, pages_t, scales in ((k, back[0], back16[0], cache.k, cache.k_scale), (v, back[1], back16[1], cache.v, cache.v_scale)):
        x64 = x.double().cpu().view(rows, heads, dh)
        got = got.cpu().view(rows, heads, dh)
        if dtype == BF16:
            want = x64.to(rows_dtype).to(BF16).double()
            assert torch.equal(got.double()[~skipped], want[~skipped])
        else:
            scale = (x64.abs().amax(-1).float().clamp(min=2.0 ** -100) / 448)
            assert torch.equal(scales.cpu()[page_of, :, at][~skipped], scale[~skipped])
            off = (got.double() - x64).abs()
            assert bool((off <= x64.abs() * (2.0 ** -4 + 4 * U) + scale[..., None] * 2.0 ** -10)[~skipped].all())
            codes = pages_t.cpu().view(torch.uint8)[page_of, :, at].view(E4M3).double()
            # the nearest code of the fp32 quotient
            want = _cast8((x64.float() / scale[..., None]).double())
            assert torch.equal(codes[~skipped], want[~skipped])
        assert bool((got[skipped] == 0).all())
        assert torch.equal(got16.cpu().view(rows, heads, dh), got.to(BF16))
    # nothing but the written slots has changed
    free = torch.ones(pages * page, dtype=torch.bool)
    free[slots.long()[~skipped]] = False
    fp, fa = torch.arange(pages * page)[free] // page, torch.arange(pages * page)[free] % page
    for now, then in zip((cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale), before):
        if now is not None:
            assert torch.equal(now.cpu()[fp, :, fa], then.cpu()[fp, :, fa])


@pytest.mark.gpu
def test_rows_of_zeros_tiny_values_and_non_finite_values():
    ops = _ops()
    cache = ops.PagedKVCache.new(1, 1, 8, 64, E4M3, DEV)
    x = torch.ones(6, 64)
    x[0] = 0.0
    x[1] = 2.0 ** -120
    x[2, 5] = math.nan
    x[3, 7] = math.inf
    x[4] = 3.3e38
    x[5, 1:] = 0.0
    slots = torch.arange(6, dtype=torch.int32, device=DEV)
    ops.kv_cache_write(cache, x.to(DEV), x.to(DEV), slots)
    k, v = (t.cpu() for t in ops.kv_cache_read(cache, slots, dtype=torch.float32))
    assert torch.equal(k[[0, 1, 4, 5]], v[[0, 1, 4, 5]])
    assert bool((k[0] == 0).all()) and bool((k[1] == 0).all())
    assert bool(k[2].isnan().all()) and bool(k[3].isnan().all())
    assert bool((k[4] / 3.3e38 - 1).abs().max() < 2.0 ** -4) and k[5, 0] == 1.0 and bool((k[5, 1:] == 0).all())


@pytest.mark.gpu
def test_rows_behind_the_slots_of_a_new_matrix_are_zeros():
    """Keys read into a given matrix with more rows than slots: its rows behind them stay, the new matrix of values has zeros."""
    ops = _ops()
    rows, slots = torch.ones(3, 2 * 64, dtype=BF16, device=DEV), torch.arange(3, dtype=torch.int32, device=DEV)
    cache = ops.PagedKVCache.new(2, 2, 16, 64, BF16, DEV)
    ops.kv_cache_write(cache, rows, rows, slots)
    for given in "kv":
        block = torch.full((50, 2 * 64), 7.0, dtype=BF16, device=DEV)
        torch.full((50, 2 * 64), 9.0, dtype=BF16, device=DEV)  # memory that held something else
        k, v = ops.kv_cache_read(cache, slots, **{given: block})
        new = v if given == "k" else k
        assert (k if given == "k" else v) is block and bool((block[3:] == 7).all())
        assert bool((k[:3] == 1).all()) and bool((v[:3] == 1).all()) and bool((new[3:] == 0).all())


# ---- attention over the cache ---------------------------------------------------------------------------------------------
def _filled(new, total, heads, page, dh, dtype, seed, cols=0, extra_pages=2):
    """A cache whose unused places hold NaN, filled through its own write; (cache, table, dense k, v [sum total, heads * dh])."""
    ops = _ops()
    g = torch.Generator().manual_seed(seed)
    need = [-(-t // page) for t in total]
    pages = sum(need) + extra_pages
    cache = ops.PagedKVCache.new(pages, heads, page, dh, dtype, DEV)
    for t in (cache.k, cache.v):
        t.view(torch.uint8).fill_(0x7f) if dtype == E4M3 else t.fill_(math.nan)
    for t in (cache.k_scale, cache.v_scale):
        if t is not None:
            t.fill_(math.nan)
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((len(total), max(max(need), 1) + cols), 1 << 30, dtype=torch.int32)  # unused entries are nobody's business
    at = 0
    slots = []
    for s, (t, m) in enumerate(zip(total, need)):
        table[s, :m] = order[at:at + m]
        slots.append(cache.slots(table[s], torch.arange(t)) if t else torch.zeros(0, dtype=torch.int32))
        at += m
    slots = torch.cat(slots).to(DEV)
    k, v = (torch.randn(max(sum(total), 1), heads * dh, generator=g).to(BF16).to(DEV) for _ in range(2))
    if sum(total):
        ops.kv_cache_write(cache, k, v, slots)
        k, v = ops.kv_cache_read(cache, slots, dtype=torch.float32)
    return cache, table.to(DEV), k[:sum(total)], v[:sum(total)]


def _paged_reference(q, k, v, new, total, Hq, Hkv, scale):
    ref = reference(q, k, v, torch.zeros_like(q), new, total, Hq, Hkv, True, scale, E16)
    p_v = reference(q, k, v.abs(), torch.zeros_like(q), new, total, Hq, Hkv, True, scale, E16)["o"][0]
    (o, tol), (lse, lse_tol) = ref["o"], ref["lse"]
    return {"o": (o, tol + 64 * U * p_v.abs()), "lse": (lse, lse_tol + 64 * U)}


PAGED = [
    # new tokens, total lengths, Hq, Hkv, page, dh
    ([1], [1], 1, 1, 8, 64),
    ([1, 1, 1, 1], [5, 300, 0, 33], 8, 8, 16, 64),            # one sequence with nothing at all
    ([1, 1, 1], [128, 257, 2000], 16, 2, 64, 128),
    ([1, 1], [9000, 700], 5, 1, 8, 64),                        # many splits of small pages
    ([5, 2, 0, 4, 3], [100, 2, 50, 1500, 3], 4, 4, 16, 128),   # drafted tokens; a sequence without new ones; a chunk that is all
    ([4, 6], [2, 40], 8, 2, 32, 64),                           # more new tokens than positions: rows that see nothing
    ([9, 5, 7], [640, 9, 333], 40, 8, 128, 64),                # 45 rows a head: two blocks of 32
    ([33, 70, 1, 20], [300, 70, 64, 1025], 8, 2, 16, 128),     # many rows
    ([200, 131], [900, 131], 3, 3, 256, 64),
    ([1] * 300, [37 * i % 1990 for i in range(300)], 2, 1, 16, 64),  # more sequences than threads, all sorts of splits
    ([1, 0, 2] * 90, [1 + 997 * i % 1500 for i in range(270)], 3, 1, 8, 128),
    # so many sequences that none is split, and one whose pages pass a window of 512
    ([1] * 20 + [3] + [1] * 43, [2] * 20 + [9001] + [5] * 43, 8, 8, 8, 64),
    ([1] * 60 + [40] + [1] * 3, [2] * 60 + [8500] + [5] * 3, 16, 8, 8, 128),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [E4M3, BF16], ids=["e4m3", "bf16"])
@pytest.mark.parametrize("case", range(len(PAGED)))
def test_paged_attention_matches_float64(case, dtype):
    ops = _ops()
    new, total, Hq, Hkv, page, dh = PAGED[case]
    cache, table, k, v = _filled(new, total, Hkv, page, dh, dtype, 60 + case, cols=case)
    ops_check = ops.check_pages
    ops_check()
    g = torch.Generator().manual_seed(case)
    wide = torch.randn(sum(new), Hq * dh + 32, generator=g).to(BF16).to(DEV)
    q = wide[:, 16:16 + Hq * dh]
    scale = 0.17
    ref = _paged_reference(q, k, v, new, total, Hq, Hkv, scale)
    lens = torch.tensor(total, dtype=torch.int32, device=DEV)
    cu = torch.tensor([0] + np.cumsum(new).tolist(), dtype=torch.int32, device=DEV)
    o, lse = ops.attn_paged(q, cache, table, lens, Hq, cu_q=cu, max_q=max(new), scale=scale, return_lse=True)
    within("o", o, ref)
    within("lse", lse, ref)
    again = ops.attn_paged(q, cache, table, lens, Hq, cu_q=cu, max_q=max(new), scale=scale)
    assert torch.equal(o, again)
    if all(a == 1 for a in new):
        single, slse = ops.attn_paged(q, cache, table, lens, Hq, scale=scale, return_lse=True)
        assert torch.equal(single, o) and torch.equal(slse, lse)
    if max(new) > 1:  # a hint that is too small is only slower
        within("o", ops.attn_paged(q, cache, table, lens, Hq, cu_q=cu, max_q=1, scale=scale), ref)
    within("o", ops.attn_paged(q, cache, table, lens, Hq, cu_q=cu, max_q=200, scale=scale), ref)
    ops_check()  # entries past a sequence's end were not even looked at


@pytest.mark.gpu
@pytest.mark.parametrize("new", [[3, 1, 2], [40, 70, 20]], ids=["few", "many"])
def test_rows_of_no_sequence_and_columns_beside_stay(new):
    ops = _ops()
    total, Hq, Hkv, dh = [500, 70, 1200], 4, 2, 64
    cache, table, k, v = _filled(new, total, Hkv, 16, dh, E4M3, 5)
    rows = sum(new) + 5
    q = torch.randn(rows, Hq * dh, generator=torch.Generator().manual_seed(2)).to(BF16).to(DEV)
    lens = torch.tensor(total, dtype=torch.int32, device=DEV)
    cu = torch.tensor([2] + (2 + np.cumsum(new)).tolist(), dtype=torch.int32, device=DEV)
    block = torch.full((rows, 3 * Hq * dh), 7.0, dtype=BF16, device=DEV)
    out = block[:, Hq * dh:2 * Hq * dh]
    ops.attn_paged(q, cache, table, lens, Hq, cu_q=cu, max_q=max(new), out=out)
    ref = _paged_reference(q[2:-3], k, v, new, total, Hq, Hkv, 0.125)
    within("o", out[2:-3], ref)
    rest = block.clone()
    rest[2:-3, Hq * dh:2 * Hq * dh] = 7
    assert bool((rest == 7).all())
    fresh = ops.attn_paged(q, cache, table, lens, Hq, cu_q=cu, max_q=max(new))
    assert torch.equal(fresh[2:-3], out[2:-3]) and bool((fresh[:2] == 0).all()) and bool((fresh[-3:] == 0).all())
    for tokens in (cu, None):  # memory that held something else, one token each as well
        torch.full((rows, Hq * dh), 9.0, dtype=BF16, device=DEV)
        fresh = ops.attn_paged(q, cache, table, lens, Hq, cu_q=tokens, max_q=max(new))
        mine = slice(2, -3) if tokens is not None else slice(0, 3)
        rest = fresh.clone()
        rest[mine] = 0
        assert bool((rest == 0).all()) and not bool((fresh[mine] == 9).any())


@pytest.mark.gpu
@pytest.mark.parametrize("new", [[1, 1, 1], [30, 50, 20]], ids=["few", "many"])
def test_bad_pages_slots_and_lengths_are_skipped_and_counted(new):
    ops = _ops()
    ops.check_pages()
    total, Hq, Hkv, dh, page = [200, 96, 70], 4, 2, 64, 16
    cache, table, k, v = _filled(new, total, Hkv, page, dh, BF16, 8)
    q = torch.randn(sum(new), Hq * dh, generator=torch.Generator().manual_seed(2)).to(BF16).to(DEV)
    cu = torch.tensor([0] + np.cumsum(new).tolist(), dtype=torch.int32, device=DEV)
    lens = torch.tensor(total, dtype=torch.int32, device=DEV)
    # sequence 1 without its third page: its positions are unseen, the later ones stay where they are
    table[1, 2] = cache.pages
    got = ops.attn_paged(q, cache, table, lens, Hq, cu_q=cu, max_q=max(new))
    with pytest.raises(IndexError):
        ops.check_pages()
    ops.check_pages()
    keep = torch.ones(total[1], dtype=torch.bool)
    keep[2 * page:3 * page] = False
    a = total[0]
    k1, v1 = k[a:a + total[1]][keep.to(DEV)], v[a:a + total[1]][keep.to(DEV)]
    # the rows of sequence 1 all lie behind the missing page
    first = total[1] - new[1]
    ref = _paged_reference(q[cu[1]:cu[2]], k1, v1, [new[1]], [total[1] - page], Hq, Hkv, 0.125) if first >= 3 * page - 1 else None
    if ref is None:
        qs = q[cu[1]:cu[2]]
        part = 3 * page - first  # rows that end on the missing page see the two pages before it at most
        late = _paged_reference(qs[part:], k1, v1, [new[1] - part], [total[1] - page], Hq, Hkv, 0.125)
        within("o", got[cu[1] + part:cu[2]], late)
    else:
        within("o", got[cu[1]:cu[2]], ref)
    assert bool(got.isfinite().all())
    # a length past the table is cut to it
    cols = table.shape[1]
    table[1, 2] = 0
    long = lens.clone()
    long[0] = cols * page + 1
    ops.attn_paged(q, cache, table, long, Hq, cu_q=cu, max_q=max(new))
    with pytest.raises(IndexError):
        ops.check_pages()
    # offsets past the rows are cut too
    wild = torch.tensor([0, new[0], 1 << 30, -5], dtype=torch.int32, device=DEV)
    ops.attn_paged(q, cache, table, lens, Hq, cu_q=wild, max_q=max(new))
    # slots past the cache: skipped when written, zeros when read
    slots = torch.tensor([0, cache.pages * page, 1], dtype=torch.int32, device=DEV)
    before = cache.k.clone()
    rows = torch.ones(3, Hkv * dh, dtype=BF16, device=DEV)
    ops.kv_cache_write(cache, rows, rows, slots)
    back, _ = ops.kv_cache_read(cache, slots)
    assert bool((back[0] == 1).all()) and bool((back[1] == 0).all()) and bool((back[2] == 1).all())
    now = cache.k.clone()
    now[0, :, :2] = before[0, :, :2]
    assert torch.equal(now.view(torch.int16), before.view(torch.int16))
    with pytest.raises(IndexError):
        ops.check_pages()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,heads,page,entry", [(1000, 1, 16, 50), (4200, 64, 8, 520)], ids=["split", "window"])
def test_bad_pages_that_only_later_rows_see_are_counted(tokens, heads, page, entry):
    """A whole prompt at once: its first tile of rows neither sees the later splits of the keys nor the later windows of pages."""
    ops = _ops()
    ops.check_pages()
    dh = 64
    cache, table, _, _ = _filled([tokens], [tokens], heads, page, dh, BF16, 12)
    q = torch.randn(tokens, heads * dh, generator=torch.Generator().manual_seed(3)).to(BF16).to(DEV)
    lens, cu = (torch.tensor(t, dtype=torch.int32, device=DEV) for t in ([tokens], [0, tokens]))
    whole = ops.attn_paged(q, cache, table, lens, heads, cu_q=cu, max_q=tokens)
    ops.check_pages()
    table[0, entry] = -1
    got = ops.attn_paged(q, cache, table, lens, heads, cu_q=cu, max_q=tokens)
    with pytest.raises(IndexError):
        ops.check_pages()
    first = entry * page
    assert torch.equal(got[:first], whole[:first]) and not torch.equal(got[first:], whole[first:]) and bool(got.isfinite().all())


@pytest.mark.gpu
def test_slots_of_positions_and_pages_that_do_not_exist():
    ops = _ops()
    ops.check_pages()
    cache = ops.PagedKVCache.new(6, 2, 16, 64, BF16, DEV)
    table = torch.tensor([3, -1, 6, 1 << 28, 5], dtype=torch.int32)
    positions = torch.tensor([0, 15, 16, 40, 48, 63, 64, 79, 80, 1 << 40, -1], dtype=torch.int64)
    none = cache.pages * cache.page
    want = [48, 63, none, none, none, none, 80, 95, none, none, none]
    for t in (table, table.to(DEV)):
        got = cache.slots(t, positions.to(t.device))
        assert got.dtype == torch.int32 and got.tolist() == want
    assert cache.slots(table[:0], positions).tolist() == [none] * len(want)
    rows = torch.ones(len(want), 2 * 64, dtype=BF16, device=DEV)
    before = cache.k.clone()
    ops.kv_cache_write(cache, rows, rows, got)
    assert torch.equal(cache.k[[0, 1, 2, 4]].view(torch.int16), before[[0, 1, 2, 4]].view(torch.int16))
    with pytest.raises(IndexError):
        ops.check_pages()


@pytest.mark.gpu
def test_counts_wait_for_work_on_other_streams():
    ops = _ops()
    ops.check_pages()
    cache = ops.PagedKVCache.new(6, 2, 16, 64, BF16, DEV)
    rows = torch.ones(3, 2 * 64, dtype=BF16, device=DEV)
    slots = torch.tensor([0, 6 * 16, 1], dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        ops.kv_cache_write(cache, rows, rows, slots)
    with pytest.raises(IndexError):
        ops.check_pages()
    ops.check_pages()


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Pages whose byte offsets pass 2^33, and packed rows 2^24 elements apart."""
    ops = _ops()
    Hkv, page, dh, pages = 4, 64, 128, (1 << 17) + 40
    cache = ops.PagedKVCache.new(pages, Hkv, page, dh, BF16, DEV)
    total, new, Hq = [300, 129], [3, 1], 8
    table = torch.zeros(2, 5, dtype=torch.int32)
    table[0], table[1, :3] = torch.arange(pages - 1, pages - 6, -1), torch.tensor([7, pages - 9, pages - 20])
    slots = torch.cat([cache.slots(table[s], torch.arange(t)) for s, t in enumerate(total)]).to(DEV)
    g = torch.Generator().manual_seed(4)
    k, v = (torch.randn(sum(total), Hkv * dh, generator=g).to(BF16).to(DEV) for _ in range(2))
    ops.kv_cache_write(cache, k, v, slots)
    back = ops.kv_cache_read(cache, slots)
    assert torch.equal(back[0], k) and torch.equal(back[1], v)
    q = torch.randn(sum(new), Hq * dh, generator=g).to(BF16).to(DEV)
    lens, cu = torch.tensor(total, dtype=torch.int32, device=DEV), torch.tensor([0, 3, 4], dtype=torch.int32, device=DEV)
    for hint in (3, 100):
        within("o", ops.attn_paged(q, cache, table.to(DEV), lens, Hq, cu_q=cu, max_q=hint),
               _paged_reference(q, k, v, new, total, Hq, Hkv, 1 / math.sqrt(dh)))
    del cache
    lq, heads, dh = [260, 30], 1, 64
    big = torch.empty(290 * (1 << 24), dtype=BF16, device=DEV)
    view = lambda at: big.as_strided((290, dh), (1 << 24, 1), at * 128)
    q, k, v, do, o, dq, dk, dv = (view(i) for i in range(8))
    for t in (q, k, v, do):
        t.copy_(torch.randn(290, dh, generator=g))
    seqs = ops.PackedSeqs(lq, device=DEV)
    _, lse = ops.attn_packed_fwd(q, k, v, heads, heads, seqs, out=o)
    ops.attn_packed_bwd(q, k, v, o, do, lse, heads, heads, seqs, dq=dq, dk=dk, dv=dv)
    ref = reference(q, k, v, do, lq, lq, heads, heads, True, 0.125, E16)
    for n, t in (("o", o), ("dq", dq), ("dk", dk), ("dv", dv)):
        within(n, t, ref)


@pytest.mark.gpu
def test_captured_steps_follow_the_tables():
    """Two captured decode steps replayed in turn, with new lengths, pages and tokens, between eager calls of other sizes."""
    ops = _ops()
    Hq, Hkv, page, dh, n = 8, 2, 16, 64, 3
    cache, table, _, _ = _filled([1] * n, [700, 650, 400], Hkv, page, dh, E4M3, 9)
    lens = torch.tensor([650, 20, 300], dtype=torch.int32, device=DEV)
    q, kn, vn = (torch.zeros(n, w * dh, dtype=BF16, device=DEV) for w in (Hq, Hkv, Hkv))
    slots = torch.zeros(n, dtype=torch.int32, device=DEV)

    def step():
        ops.kv_cache_write(cache, kn, vn, slots)
        return ops.attn_paged(q, cache, table, lens, Hq)

    step()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step())
    g = torch.Generator().manual_seed(3)
    for turn in range(4):
        for t in (q, kn, vn):
            t.copy_(torch.randn(t.shape, generator=g))
        lens.copy_(torch.tensor([651 + turn, 21 + 100 * turn, 1 + turn]))
        slots.copy_(torch.cat([cache.slots(table[s].cpu(), (lens[s:s + 1] - 1).cpu()) for s in range(n)]))
        graphs[turn % 2].replay()
        torch.cuda.synchronize()
        got = outs[turn % 2].clone()
        assert torch.equal(got, ops.attn_paged(q, cache, table, lens, Hq))
        ops.attn_paged(q[:1], cache, table[:1], lens[:1], Hq)
        torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.attn_paged(q, cache, table, lens, Hq)
    mine = ops.attn_paged(q, cache, table, lens, Hq)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(mine, other)


# ---- verification -------------------------------------------------------------------------------------------------------
def _verified(target, draft, tokens, u, us, num, pad):
    """The definition, row by row, in double."""
    n, d = tokens.shape
    V = target.shape[2]
    out, counts = np.full((n, d + 1), pad, np.int64), np.zeros(n, np.int32)
    for b in range(n):
        i = 0
        while i < num[b]:
            x = tokens[b, i]
            q = 1.0 if draft is None else (float(draft[b, i, x]) if 0 <= x < V else 0.0)
            if not (0 <= x < V and float(u[b, i]) * q < float(target[b, i, x])):
                break
            out[b, i] = x
            i += 1
        p = target[b, i].astype(np.float64)
        w = p.copy()
        if i < num[b]:
            if draft is not None:
                w = p - draft[b, i].astype(np.float64)
            elif 0 <= tokens[b, i] < V:
                w[tokens[b, i]] = 0
        w = np.where(w > 0, w, 0)
        if w.sum() <= 0:
            w = np.where(p > 0, p, 0)
        sums, some = np.cumsum(w), np.nonzero(w)[0]
        out[b, i] = min(np.searchsorted(sums, float(us[b]) * sums[-1], side="right"), some[-1]) if len(some) else 0
        counts[b] = i
    return out, counts


@pytest.mark.gpu
@pytest.mark.parametrize("sure", [False, True], ids=["draft", "sure"])
@pytest.mark.parametrize("n,d,V", [(1, 1, 1), (3, 4, 2), (7, 5, 257), (33, 3, 4099), (5, 64, 1000), (4, 2, 70001), (6, 0, 999)])
def test_drafts_are_verified(n, d, V, sure):
    ops = _ops()
    g = torch.Generator().manual_seed(n + V)
    logits = 2 * torch.randn(n, d + 1, V, generator=g)
    target = torch.softmax(logits, -1)
    draft = torch.softmax(logits[:, :d] + 0.5 * torch.randn(n, d, V, generator=g), -1)
    tokens = draft.argmax(-1)
    if n > 2 and d > 1:
        tokens[0, 0], tokens[1, 1] = -1, V      # refused
        draft[2] = target[2, :d]                # nothing left of p - q
    u, us = torch.rand(n, d, generator=g), torch.rand(n, generator=g)
    us[0] = 0.0
    us[-1] = 1 - 2.0 ** -24
    num = torch.randint(0, d + 2, (n,), generator=g).to(torch.int32)  # one too many here and there: cut
    if n > 2 and d > 1:
        num[:3] = d
    wide_t, wide_d = torch.zeros(n, d + 2, V + 5, device=DEV), torch.zeros(n, d + 1, V + 3, device=DEV)
    wide_t[:, :d + 1, :V], wide_d[:, :d, :V] = target.to(DEV), draft.to(DEV)
    for number in (num, None):
        cut = (num if number is not None else torch.full((n,), d)).clamp(0, d).numpy()
        want = _verified(target.numpy(), None if sure else draft.numpy(), tokens.numpy(), u.numpy(), us.numpy(), cut, -7)
        for t, q in ((target.to(DEV), draft.to(DEV)), (wide_t[:, :d + 1, :V], wide_d[:, :d, :V])):
            out, acc = ops.draft_verify(t, None if sure else q, tokens.to(DEV), u.to(DEV), us.to(DEV),
                                        num_draft=None if number is None else number.to(DEV), pad=-7)
            assert out.dtype == torch.int64 and acc.dtype == torch.int32
            assert np.array_equal(acc.cpu().numpy(), want[1])
            assert np.array_equal(out.cpu().numpy(), want[0])


@pytest.mark.gpu
def test_verification_edges():
    ops = _ops()
    V = 300
    target, draft = torch.zeros(4, 2, V), torch.zeros(4, 1, V)
    target[0, :, 5] = 1.0                       # certain target, the same draft: accepted with any u < 1
    draft[0, 0, 5] = 1.0
    target[1, 0, 7] = draft[1, 0, 7] = 0.5      # p = q everywhere, refused by u q = p: drawn from p
    target[1, 0, 9] = draft[1, 0, 9] = 0.5
    target[3, 0, 2], target[3, 0, 4] = math.nan, 0.25  # NaN counts as 0
    tokens = torch.tensor([[5], [7], [0], [2]])
    u, us = torch.tensor([[0.999], [1.0], [0.0], [0.0]]), torch.tensor([0.3, 0.75, 0.5, 0.99])
    out, acc = ops.draft_verify(*(t.to(DEV) for t in (target, draft, tokens, u, us)))
    assert acc.tolist() == [1, 0, 0, 0]
    assert out.tolist() == [[5, 5], [9, 0], [0, 0], [4, 0]]


def _scan(x):
    """Running sums over 64 lanes in the order of a scan by doubling distances."""
    x, o = x.copy(), 1
    while o < 64:
        x[o:] = x[o:] + x[:-o].copy()
        o *= 2
    return x


def _an_inversion():
    """256 weights with four zeros in one lane at which the scan's sum is one last bit above the lane before, that lane, and
    weights to go behind them whose total makes half of everything equal to the sum before the zeros."""
    rng = np.random.default_rng(0)
    for _ in range(20000):
        w = (rng.random(256) * 2.0 ** rng.integers(-30, 0, 256)).astype(np.float32)
        lane = int(rng.integers(2, 60))
        w[4 * lane:4 * lane + 4] = 0
        d = w.astype(np.float64).reshape(64, 4)
        mine = ((d[:, 0] + d[:, 1]) + d[:, 2]) + d[:, 3]
        upto, total = _scan(mine), mine.copy()
        for o in (32, 16, 8, 4, 2, 1):
            total = total + total[np.arange(64) ^ o]
        border = upto[lane - 1]
        rest, left = [], 2 * border - total[0]
        for _ in range(3):  # 53 bits as three numbers of 24
            rest.append(np.float32(left))
            left -= float(rest[-1])
        behind = float(rest[0]) + float(rest[1]) + float(rest[2])
        if int(np.argmax(upto > border)) == lane and left == 0 and min(rest) > 0 and total[0] + behind == 2 * border:
            return w, lane, rest
    raise AssertionError("no such weights")


@pytest.mark.gpu
def test_a_draw_on_the_border_of_tokens_without_weight():
    """The draw falls on the border to four tokens of weight zero, where a sum of another order is one last bit higher: it takes
    a neighbour of the border, not whatever token comes last."""
    ops = _ops()
    w, lane, rest = _an_inversion()
    target = torch.zeros(1, 1, 4096)
    target[0, 0, :256] = torch.from_numpy(w)
    target[0, 0, 300:303] = torch.from_numpy(np.array(rest))
    none = torch.zeros(1, 0, device=DEV)
    out, acc = ops.draft_verify(target.to(DEV), None, none.long(), none, torch.tensor([0.5], device=DEV))
    below, above = np.flatnonzero(w[:4 * lane])[-1], 4 * lane + 4 + np.flatnonzero(w[4 * lane + 4:])[0]
    assert acc.tolist() == [0] and out.item() in (below, above), (out.item(), below, above)


# ---- a program that uses them together ---------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [E4M3, BF16], ids=["e4m3", "bf16"])
def test_prompt_cache_drafts_and_verification_together(dtype):
    """Prompts through packed attention, their keys and values into the cache, then steps of drafted tokens: written, attended
    over the cache, verified, and the lengths moved on by what was accepted; every attention output is checked against float64
    over what the cache is meant to hold at that time."""
    ops = _ops()
    Hq, Hkv, dh, page, drafts, V = 8, 2, 64, 16, 3, 500
    g = torch.Generator().manual_seed(77)
    prompts = [35, 1, 130]
    n = len(prompts)
    cache = ops.PagedKVCache.new(40, Hkv, page, dh, dtype, DEV)
    table = torch.randperm(40, generator=g)[:n * 12].view(n, 12).to(torch.int32)
    q, k, v = (torch.randn(sum(prompts), w * dh, generator=g).to(BF16).to(DEV) for w in (Hq, Hkv, Hkv))
    o, _ = ops.attn_packed_fwd(q, k, v, Hq, Hkv, ops.PackedSeqs(prompts, device=DEV))
    within("o", o, reference(q, k, v, torch.zeros_like(q), prompts, prompts, Hq, Hkv, True, 0.125, E16))
    slots = torch.cat([cache.slots(table[s], torch.arange(t)) for s, t in enumerate(prompts)])
    ops.kv_cache_write(cache, k, v, slots.to(DEV))
    held = list(ops.kv_cache_read(cache, slots.to(DEV), dtype=torch.float32))
    held = [[t.cpu() for t in x.split(prompts)] for x in held]  # what the cache is meant to hold, sequence by sequence
    lens = list(prompts)
    head = torch.randn(Hq * dh, V, generator=g).to(DEV)
    for step in range(4):
        new = [drafts + 1 if s != step % n else 2 for s in range(n)]  # one sequence drafts a single token
        rows = sum(new)
        q, k, v = (torch.randn(rows, w * dh, generator=g).to(BF16).to(DEV) for w in (Hq, Hkv, Hkv))
        total = [a + b for a, b in zip(lens, new)]
        slots = torch.cat([cache.slots(table[s], torch.arange(lens[s], total[s])) for s in range(n)]).to(DEV)
        ops.kv_cache_write(cache, k, v, slots)
        back = [t.cpu().split(new) for t in ops.kv_cache_read(cache, slots, dtype=torch.float32)]
        held = [[torch.cat([old[:lens[s]], x[s]]) for s, old in enumerate(side)] for side, x in zip(held, back)]
        cu = torch.tensor([0] + np.cumsum(new).tolist(), dtype=torch.int32, device=DEV)
        o = ops.attn_paged(q, cache, table.to(DEV), torch.tensor(total, dtype=torch.int32, device=DEV), Hq, cu_q=cu, max_q=drafts + 1)
        within("o", o, _paged_reference(q, torch.cat(held[0]), torch.cat(held[1]), new, total, Hq, Hkv, 0.125))
        target = torch.zeros(n, drafts + 1, V, device=DEV)
        for s in range(n):
            target[s, :new[s]] = torch.softmax(o[cu[s]:cu[s + 1]].float() @ head * 0.3, -1)
        near = torch.softmax(torch.log(target[:, :drafts] + 1e-9) + 0.3 * torch.randn(n, drafts, V, generator=g).to(DEV), -1)
        tokens = near.argmax(-1)
        u, us = torch.rand(n, drafts, generator=g), torch.rand(n, generator=g)
        num = torch.tensor([a - 1 for a in new], dtype=torch.int32)
        out, acc = ops.draft_verify(target, near, tokens, u.to(DEV), us.to(DEV), num_draft=num.to(DEV))
        want = _verified(target.cpu().numpy(), near.cpu().numpy(), tokens.cpu().numpy(), u.numpy(), us.numpy(), num.numpy(), 0)
        assert np.array_equal(out.cpu().numpy(), want[0]) and np.array_equal(acc.cpu().numpy(), want[1])
        lens = [a + 1 + int(c) for a, c in zip(lens, acc.cpu())]  # refused tokens are overwritten by the next step
    ops.check_pages()


# ---- refusals -------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_calls_on_two_streams_at_once():
    """Calls with scratch of their own (split keys, walks in parts), overlapping on two streams."""
    ops = _ops()
    g = torch.Generator().manual_seed(3)
    works = []
    for i in range(2):
        total = [3000 + 500 * i, 700, 90]
        cache, table, _, _ = _filled([2, 1, 3], total, 2, 16, 128, (BF16, E4M3)[i], 900 + i)
        q = torch.randn(6, 8 * 128, generator=g).to(BF16).to(DEV)
        lens, cu = torch.tensor(total, dtype=torch.int32, device=DEV), torch.tensor([0, 2, 3, 6], dtype=torch.int32, device=DEV)
        lengths = [1200 + 100 * i, 33]
        wide = torch.randn(sum(lengths), 4 * 256, generator=g).to(BF16).to(DEV)
        seqs = ops.PackedSeqs(lengths, device=DEV)

        def work(cache=cache, table=table, q=q, lens=lens, cu=cu, wide=wide, seqs=seqs):
            o, lse = ops.attn_packed_fwd(wide[:, :256], wide[:, 256:320], wide[:, 320:384], 4, 1, seqs)
            grads = ops.attn_packed_bwd(wide[:, :256], wide[:, 256:320], wide[:, 320:384], o, wide[:, 512:768], lse, 4, 1, seqs)
            return [o, *grads, ops.attn_paged(q, cache, table, lens, 8, cu_q=cu, max_q=3)]

        works.append(work)
    want = [w() for w in works]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in works]
    got = []
    for turn in range(6):
        for w, s in zip(works, streams):
            with torch.cuda.stream(s):
                got.append(w())
    torch.cuda.synchronize()
    for i, res in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(res, want[i % 2])), i


@pytest.mark.gpu
def test_direct_and_general_calls_agree(monkeypatch):
    """The direct calls (csrc/calls.cpp) take the plain forms and do what the general way through ctypes does."""
    from imagecaption_amd import _capi
    ops = _ops()
    _capi.lib()
    assert _capi.fast is not None
    g = torch.Generator().manual_seed(7)
    rand = lambda *shape, dtype=BF16: torch.randn(*shape, generator=g).to(dtype).to(DEV)
    taken = []

    class Counted:
        def __getattr__(self, name):
            call = getattr(direct, name)

            def counted(*args):
                done = call(*args)
                taken.append((name, done is not None))
                return done
            return counted

    direct = _capi.fast
    seqs = {n: ops.PackedSeqs(lens, device=DEV) for n, lens in (("long", [70, 200, 1]), ("short", [9, 20, 32]))}
    wide = rand(271, 3 * 256)
    probs = torch.rand(3, 4, 50, generator=g).to(DEV)
    tokens, u, us = torch.randint(0, 50, (3, 3), generator=g).to(DEV), torch.rand(3, 3, generator=g).to(DEV), torch.rand(3, generator=g).to(DEV)
    table = torch.arange(12, dtype=torch.int32).view(3, 4).to(DEV)
    lens, cu = torch.tensor([60, 3, 17], dtype=torch.int32, device=DEV), torch.tensor([0, 2, 3, 6], dtype=torch.int32, device=DEV)

    def everything():
        out = []
        for dtype in (BF16, torch.float32):
            for name, rows in (("long", 271), ("short", 61)):
                x = wide[:rows].to(dtype)
                q, k, v = x[:, :256], x[:, 256:384], x[:, 384:512]
                for scale in (None, 0.3):
                    o, lse = ops.attn_packed_fwd(q, k, v, 4, 2, seqs[name], scale=scale)
                    out += [o, lse, *ops.attn_packed_bwd(q, k, v, o, x[:, 512:], lse, 4, 2, seqs[name], scale=scale)]
                o, lse = ops.attn_packed_fwd(q, k, v, 4, 2, seqs[name], save_lse=False)
                assert lse is None
                out.append(o)
        for dtype in (BF16, E4M3):
            cache = ops.PagedKVCache(*(torch.zeros(12, 2, 16, 64, dtype=torch.uint8 if dtype == E4M3 else dtype, device=DEV).view(dtype)
                                       for _ in range(2)),
                                     *((torch.zeros(12, 2, 16, device=DEV) for _ in range(2)) if dtype == E4M3 else ()))
            slots = torch.arange(192, dtype=torch.int32, device=DEV)
            ops.kv_cache_write(cache, wide[:192, :128], wide[:192, 128:256], slots)
            ops.kv_cache_write(cache, wide[:5, :128].float(), wide[:5, 128:256].float(), slots[100:105])
            out += [*ops.kv_cache_read(cache, slots), *ops.kv_cache_read(cache, slots[7:8], dtype=torch.float32)]
            out += [ops.attn_paged(wide[:6, :256], cache, table, lens, 4, cu_q=cu, max_q=3),
                    ops.attn_paged(wide[:5, :512], cache, table, lens, 8, scale=0.2)]
        out += [*ops.draft_verify(probs, probs[:, 1:], tokens, u, us, pad=-1), *ops.draft_verify(probs, None, tokens, u, us, num_draft=lens)]
        return out

    monkeypatch.setattr(_capi, "fast", Counted())
    with_direct = everything()
    assert all(done for _, done in taken) and {n for n, _ in taken} == {"attn_packed_fwd", "attn_packed_bwd", "kv_cache_write", "kv_cache_read",
                                                                        "attn_paged", "draft_verify"}
    monkeypatch.setattr(_capi, "fast", None)
    general = everything()
    assert len(general) == len(with_direct) and all(a.dtype == b.dtype and torch.equal(a, b) for a, b in zip(general, with_direct))


def test_direct_calls_leave_what_they_do_not_know():
    from imagecaption_amd import _capi
    _capi.lib()
    if _capi.fast is None:
        pytest.skip("the direct calls are not built")
    x, y = torch.zeros(3, 64), [None] * 12
    assert _capi.fast.attn_packed_fwd(*y[:10]) is None and _capi.fast.attn_packed_bwd(*y) is None and _capi.fast.kv_cache_write(*y[:6]) is None
    assert _capi.fast.kv_cache_read(*y[:5]) is None and _capi.fast.attn_paged(*y[:10]) is None and _capi.fast.draft_verify(*y[:9]) is None
    assert _capi.fast.draft_verify(x, None, x, x, x, None, 0, 0, 0) is None and _capi.fast.kv_cache_write() is None
    with pytest.raises(TypeError):
        _capi.fast.bind(1, 2)


def test_arguments_are_refused_without_a_gpu():
    from imagecaption_amd import _capi
    from imagecaption_amd._capi import CapdecError
    ops = _ops()
    with pytest.raises(CapdecError, match="no CPU fallback"):
        ops.PagedKVCache(torch.zeros(2, 1, 8, 64, dtype=BF16), torch.zeros(2, 1, 8, 64, dtype=BF16))
    with pytest.raises(CapdecError, match="no CPU fallback"):
        ops.draft_verify(torch.zeros(1, 1, 4), None, torch.zeros(1, 0, dtype=torch.int64), torch.zeros(1, 0), torch.zeros(1))
    lib = _capi.lib()
    good = dict(k=16, v=16, k_scale=None, v_scale=None, pages=4, heads=2, page=16, dh=64, dtype=_capi.BF16S)

    def cache(**change):
        return C.byref(_capi.KVCache(*dict(good, **change).values()))

    bad = (dict(k=None), dict(v=8), dict(pages=0), dict(heads=0), dict(page=12), dict(page=4), dict(page=512), dict(dh=32), dict(dtype=0),
           dict(dtype=_capi.E4M3), dict(pages=1 << 28, page=8))
    for change in bad:
        assert lib.capdec_kv_write(cache(**change), 16, 128, 16, 128, 0, 16, 3, None) == -1, change
        assert lib.capdec_kv_read(cache(**change), 16, 3, 16, 128, 16, 128, 0, None) == -1, change
        assert lib.capdec_attn_paged(cache(**change), 16, 128, None, 16, 16, 4, 4, 3, 3, 1, 2, 0.1, 16, 128, 0, None, None, 0, None) == -1, change
        assert lib.capdec_attn_paged_workspace_bytes(cache(**change), 3, 3, 1, 2, 4) == 0
    for k, ldk, v, ldv, dtype, slots, rows in ((None, 128, 16, 128, 0, 16, 3), (16, 64, 16, 128, 0, 16, 3), (16, 130, 16, 128, 0, 16, 3),
                                                (16, 128, 8, 128, 0, 16, 3), (16, 128, 16, 128, 1, 16, 3), (16, 128, 16, 128, 0, None, 3),
                                                (16, 128, 16, 128, 0, 16, -1), (16, 132, 16, 128, 3, 16, 3)):
        assert lib.capdec_kv_write(cache(), k, ldk, v, ldv, dtype, slots, rows, None) == -1
    assert lib.capdec_kv_write(cache(), None, 0, None, 0, 0, None, 0, None) == 0  # no rows: nothing to do
    args = dict(q=16, ldq=128, cu=None, lens=16, table=16, ld=4, cols=4, n=3, rows=3, max_q=1, Hq=2, scale=0.1, o=16, ldo=128, clear=0, lse=None,
                ws=None, wb=0, st=None)
    for change in (dict(q=None), dict(ldq=64), dict(ldq=130), dict(lens=None), dict(table=None), dict(ld=3), dict(cols=0), dict(n=0),
                   dict(rows=2), dict(rows=-1), dict(max_q=0), dict(Hq=3), dict(Hq=0), dict(scale=0.0), dict(scale=math.inf), dict(o=8),
                   dict(ldo=100)):
        assert lib.capdec_attn_paged(cache(), *dict(args, **change).values()) == -1, change
    # a long table is split, and then needs its workspace
    need = lib.capdec_attn_paged_workspace_bytes(cache(pages=4096), 3, 3, 1, 2, 4096)
    assert need > 0
    assert lib.capdec_attn_paged(cache(pages=4096), *dict(args, cols=4096, ld=4096).values()) == -1
    assert lib.capdec_attn_paged(cache(pages=4096), *dict(args, cols=4096, ld=4096, ws=16, wb=need - 1).values()) == -4
    v = dict(t=16, ts=100, tr=50, d=16, ds=100, dr=50, tok=16, ldt=2, num=None, u=16, ldu=2, us=16, n=2, drafts=2, V=50, pad=0, out=16, acc=16, st=None)
    for change in (dict(t=None), dict(tr=49), dict(dr=49), dict(tok=None), dict(ldt=1), dict(u=None), dict(ldu=1), dict(us=None), dict(n=-1),
                   dict(drafts=65), dict(drafts=-1), dict(V=0), dict(out=None), dict(acc=None)):
        assert lib.capdec_draft_verify(*dict(v, **change).values()) == -1, change
    assert lib.capdec_draft_verify(*dict(v, n=0).values()) == 0


@pytest.mark.gpu
def test_tensors_that_do_not_fit_are_refused():
    from imagecaption_amd._capi import CapdecError
    ops = _ops()
    cache, table, k, v = _filled([1, 1], [20, 9], 2, 16, 64, E4M3, 1)
    q, lens = torch.zeros(2, 256, dtype=BF16, device=DEV), torch.tensor([20, 9], dtype=torch.int32, device=DEV)
    ops.attn_paged(q, cache, table, lens, 4)
    for args in ((q.float(), cache, table, lens, 4), (q[:1], cache, table, lens, 4), (q, cache, table.long(), lens, 4),
                 (q, cache, table[:1], lens, 4), (q, cache, table.t(), lens, 4), (q, cache, table, lens.long(), 4), (q, cache, table, lens, 3),
                 (q[:, :192], cache, table, lens, 3), (q.cpu(), cache, table, lens, 4)):
        with pytest.raises(CapdecError):
            ops.attn_paged(*args)
    for kw in (dict(max_q=0), dict(scale=0.0), dict(scale=math.nan), dict(cu_q=lens), dict(out=torch.zeros(2, 256, device=DEV))):
        with pytest.raises(CapdecError):
            ops.attn_paged(q, cache, table, lens, 4, **kw)
    rows, slots = torch.zeros(2, 128, dtype=BF16, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    for args in ((rows.half(), rows.half(), slots), (rows, rows.float(), slots), (rows[:1], rows[:1], slots), (rows[:, :64], rows, slots),
                 (rows, rows, slots.long()), (rows, rows, slots.cpu())):
        with pytest.raises(CapdecError):
            ops.kv_cache_write(cache, *args)
    for bad in ((cache.k, cache.v), (cache.k, cache.v, cache.k_scale[:1], cache.v_scale), (cache.k[:, :, :12], cache.v[:, :, :12], None, None),
                (cache.k.float(), cache.v.float())):
        with pytest.raises(CapdecError):
            ops.PagedKVCache(*bad)
    with pytest.raises(CapdecError):
        ops.PagedKVCache.new(2, 1, 24, 64, BF16, DEV)
    p = torch.rand(2, 3, 50, device=DEV)
    tok, u, us = torch.zeros(2, 2, dtype=torch.int64, device=DEV), torch.rand(2, 2, device=DEV), torch.rand(2, device=DEV)
    ops.draft_verify(p, p[:, :2], tok, u, us)
    for args in ((p.double(), p[:, :2], tok, u, us), (p, p, tok, u, us), (p, p[:, :2], tok.int(), u, us), (p, p[:, :2], tok[:1], u, us),
                 (p, p[:, :2], tok, u[:, :1], us), (p, p[:, :2], tok, u, us[:1]), (p.transpose(1, 2), None, tok, u, us),
                 (p[0], p[0], tok, u, us), (p, p[:, :2].half(), tok, u, us)):
        with pytest.raises(CapdecError):
            ops.draft_verify(*args)
    with pytest.raises(CapdecError):
        ops.draft_verify(p, p[:, :2], tok, u, us, num_draft=torch.zeros(3, dtype=torch.int32, device=DEV))


@pytest.mark.gpu
def test_pages_are_not_checked_under_capture():
    """The check reads counters on the host: refused while a graph is captured, and the capture goes on."""
    from imagecaption_amd._capi import CapdecError
    ops = _ops()
    ops.check_pages()
    x = torch.zeros(4, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x += 1
        with pytest.raises(CapdecError, match="captured"):
            ops.check_pages()
        x += 1
    for turn in range(1, 4):
        graph.replay()
        assert x.tolist() == [2.0 * turn] * 4
    ops.check_pages()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [E4M3, BF16], ids=["e4m3", "bf16"])
@pytest.mark.parametrize("new", [[1, 2, 1], [40, 70, 20]], ids=["few", "many"])
def test_scores_up_to_the_documented_size_stay_finite(new, dtype):
    ops = _ops()
    total, Hq, Hkv = [700, 70, 1200], 4, 2
    cache, table, k, _ = _filled(new, total, Hkv, 16, 64, dtype, 14)
    q = torch.randn(sum(new), Hq * 64, generator=torch.Generator().manual_seed(4)).to(BF16).to(DEV)
    top = max(float((a.float() @ b.float().T).abs().max()) for a in q.split(64, 1) for b in k.split(64, 1))
    lens, cu = (torch.tensor(t, dtype=torch.int32, device=DEV) for t in (total, [0] + np.cumsum(new).tolist()))
    o, lse = ops.attn_paged(q, cache, table, lens, Hq, cu_q=cu, max_q=max(new), scale=2.0 ** 24 / top, return_lse=True)
    assert bool(o.isfinite().all()) and bool(lse.isfinite().all()) and float(lse.abs().max()) > 2.0 ** 20


def test_pages_are_checked_where_there_is_a_gpu():
    from imagecaption_amd._capi import CapdecError
    if torch.cuda.is_available():
        pytest.skip("there is a GPU")
    with pytest.raises(CapdecError):
        _ops().check_pages()
