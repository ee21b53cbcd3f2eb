"""Attention over packed sequences (ops.attn_packed_fwd / _bwd, functional.attn_packed) against the formulas in float64.

Tolerances are worst cases, element by element, computed beside the reference.  With u = 2^-24 (fp32) and e = 2^-8 (bf16,
half a step relative to the value; 0 for fp32 matrices):
* a score is a sum of dh products: |ds| <= (dh + 4) u scale |q|.|k|, and a weight's relative error is w = 2 max|ds| + 16 u
  (exponential, its argument, lse);
* o = sum p v: (w + (nk + 8) u + e) sum p |v|, plus the result's own rounding e |o| (u |o|);
* dv the same with do; score gradients ds = p (dp - delta): delta comes from the rounded o, so its error is do (o's tolerance)
  plus sums, dp is a sum of dh products; the rounding of ds costs e |ds|; dq, dk sum these against |k|, |q|.
"""
import ctypes as C
import math

import pytest
import torch

DEV = "cuda"
U, E16 = 2.0 ** -24, 2.0 ** -8


def _ops():
    from imagecaption_amd import ops
    return ops


def reference(q, k, v, do, lq, lk, Hq, Hkv, causal, scale, e):
    """Float64 results and tolerances of every output, as {name: (value, tolerance)}."""
    dh, group = q.shape[1] // Hq, Hq // Hkv
    q, k, v, do = (t.detach().double().cpu() for t in (q, k, v, do))
    val = {n: torch.zeros_like(t) for n, t in (("o", q), ("dq", q), ("dk", k), ("dv", v))}
    tol = {n: torch.zeros_like(t) for n, t in val.items()}
    val["lse"] = torch.full((Hq, q.shape[0]), -math.inf, dtype=torch.float64)
    tol["lse"] = torch.zeros_like(val["lse"])
    a = b = 0
    for nq, nk in zip(lq, lk):
        for h in range(Hq):
            rq, rk = slice(a, a + nq), slice(b, b + nk)
            cq, ck = slice(h * dh, (h + 1) * dh), slice(h // group * dh, (h // group + 1) * dh)
            Q, K, V, D = q[rq, cq], k[rk, ck], v[rk, ck], do[rq, cq]
            s = Q @ K.T * scale
            seen = torch.ones(nq, nk, dtype=torch.bool)
            if causal:
                seen = torch.arange(nk)[None, :] <= torch.arange(nq)[:, None] + nk - nq
            s = s.masked_fill(~seen, -math.inf)
            lse = torch.logsumexp(s, 1) if nk else torch.full((nq,), -math.inf, dtype=torch.float64)
            p = torch.where(seen, torch.exp(s - torch.where(lse.isinf(), 0.0, lse)[:, None]), 0.0)
            big = float((Q.abs() @ K.abs().T).max()) * scale if nk and nq else 0.0
            w = 2 * (dh + 4) * U * big + 16 * U
            up = max(e, U)
            o = p @ V
            o_tol = (w + (nk + 8) * U + e) * (p @ V.abs()) + up * o.abs()
            val["o"][rq, cq], tol["o"][rq, cq] = o, o_tol
            val["lse"][h, rq] = lse
            tol["lse"][h, rq] = w + (nk + 8) * U + 4 * U * torch.where(lse.isinf(), 0.0, lse).abs()
            delta = (D * o).sum(1, keepdim=True)
            d_delta = (D.abs() * o_tol).sum(1, keepdim=True) + (dh + 4) * U * (D * o).abs().sum(1, keepdim=True)
            dp = D @ V.T
            d_dp = (dh + 4) * U * (D.abs() @ V.abs().T)
            ds = p * (dp - delta)
            d_ds = p * (d_dp + d_delta) + (w + e + 4 * U) * p * (dp.abs() + delta.abs())
            dv, dk, dq = p.T @ D, ds.T @ Q * scale, ds @ K * scale
            val["dq"][rq, cq] = dq
            tol["dq"][rq, cq] = scale * ((d_ds + (nk + 8) * U * ds.abs()) @ K.abs()) + up * dq.abs()
            val["dk"][rk, ck] += dk
            val["dv"][rk, ck] += dv
            tol["dk"][rk, ck] += scale * ((d_ds + (group * nq + 8) * U * ds.abs()).T @ Q.abs())
            tol["dv"][rk, ck] += (w + (group * nq + 8) * U + e) * (p.T @ D.abs())
        a, b = a + nq, b + nk
    for n in ("dk", "dv"):
        tol[n] += max(e, U) * val[n].abs()
    return {n: (val[n], tol[n]) for n in val}


def within(name, got, ref, rows=None):
    val, tol = ref[name]
    got = got.detach().double().cpu()
    assert got.shape == val.shape, (name, got.shape, val.shape)
    same = (got == val)  # -inf of empty rows
    off = torch.where(same, 0.0, (got - val).abs())
    assert bool((off <= tol * 1.001 + 1e-30).all()), (name, float((off / (tol + 1e-30)).max()), float(off.max()))


CASES = [
    # lengths of queries, of keys (None: the same), causal, Hq, Hkv, dh
    ([1], None, True, 1, 1, 64),
    ([0, 5, 0, 33, 1], None, True, 4, 2, 64),
    ([20, 8, 13, 20, 9, 17, 1], None, True, 8, 8, 64),
    ([32, 31, 33, 64, 65], None, True, 6, 2, 128),
    ([129, 300, 128, 127, 1], None, True, 8, 1, 64),
    ([200, 385], None, True, 5, 5, 128),
    ([257, 130], None, False, 8, 2, 64),
    ([20, 3, 17], [49, 49, 196], False, 8, 8, 64),
    ([5, 40, 200, 7], [0, 3, 150, 7], True, 2, 1, 64),     # rows that see nothing: no keys, fewer keys than queries
    ([5, 140, 33], [70, 300, 0], True, 4, 4, 128),         # new rows at the end of longer key sequences
    ([0, 0, 0], [3, 0, 140], False, 2, 2, 64),             # keys nobody looks at: zero gradients
]


def _inputs(lq, lk, Hq, Hkv, dh, dtype, seed, extra=0):
    """Column slices of one over-wide block for each side, with `extra` rows behind the last sequence."""
    g = torch.Generator().manual_seed(seed)
    rq, rk = sum(lq) + extra, sum(lk) + extra
    wide = torch.randn(max(rq, 1), 2 * Hq * dh + 16, generator=g).to(dtype).to(DEV)
    kv = torch.randn(max(rk, 1), 2 * Hkv * dh + 8, generator=g).to(dtype).to(DEV)
    q, do = wide[:rq, 8:8 + Hq * dh], wide[:rq, 16 + Hq * dh:]
    return q, kv[:rk, :Hkv * dh], kv[:rk, 8 + Hkv * dh:], do


@pytest.mark.gpu
@pytest.mark.parametrize("lq, lk, causal, Hq, Hkv, dh", [
    ([70, 33, 128, 127] * 6, None, True, 8, 4, 64), ([70, 33, 128, 127] * 6, [40, 100, 0, 65] * 6, False, 8, 2, 128),  # 64 rows a workgroup
    ([130, 257, 128, 40] * 7 + [1], None, True, 8, 4, 128), ([130, 257, 128, 40] * 7, [70, 300, 1, 0] * 7, True, 8, 8, 64),  # 128 rows
    ([129, 200] * 12, [65, 31] * 12, False, 8, 1, 128)])
def test_heights_of_workgroups_match_float64(lq, lk, causal, Hq, Hkv, dh):
    """Batches with enough tiles for the taller workgroups of bf16 matrices."""
    ops = _ops()
    q, k, v, do = _inputs(lq, lk or lq, Hq, Hkv, dh, torch.bfloat16, 700 + dh)
    scale = 1 / math.sqrt(dh)
    ref = reference(q, k, v, do, lq, lk or lq, Hq, Hkv, causal, scale, E16)
    seqs = ops.PackedSeqs(lq, lk, causal=causal, device=DEV)
    assert seqs.c.tiles[1] * Hq >= 256 and (seqs.c.tiles[0] * Hq >= 320) == (max(lq) > 128)
    o, lse = ops.attn_packed_fwd(q, k, v, Hq, Hkv, seqs)
    within("lse", lse, ref)
    grads = ops.attn_packed_bwd(q, k, v, o, do, lse, Hq, Hkv, seqs)
    for name, t in zip(("o", "dq", "dk", "dv"), (o, *grads)):
        within(name, t, ref)
    assert all(torch.equal(a, b) for a, b in zip(grads, ops.attn_packed_bwd(q, k, v, o, do, lse, Hq, Hkv, seqs)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lq, lk, causal, Hq, Hkv, dh", [([1500, 70], None, True, 8, 1, 64), ([900, 40, 1], [300, 7, 1000], False, 6, 2, 128),
                                                         ([1100] + [65] * 30, None, True, 4, 4, 128)])
def test_long_walks_in_parts_match_float64(dtype, lq, lk, causal, Hq, Hkv, dh):
    """Key tiles whose sums over the queries are cut into parts."""
    from imagecaption_amd import _capi
    ops = _ops()
    q, k, v, do = _inputs(lq, lk or lq, Hq, Hkv, dh, dtype, 500 + dh)
    scale = 1 / math.sqrt(dh)
    ref = reference(q, k, v, do, lq, lk or lq, Hq, Hkv, causal, scale, E16 if dtype == torch.bfloat16 else 0.0)
    seqs = ops.PackedSeqs(lq, lk, causal=causal, device=DEV)
    stats = (16 if dtype == torch.bfloat16 else 4) * Hq * sum(lq) + 15
    assert _capi.lib().capdec_attn_packed_scratch_bytes(seqs.cref, sum(lq), Hq, Hkv, dh, _capi.BF16S if dtype == torch.bfloat16 else 0) > stats
    o, lse = ops.attn_packed_fwd(q, k, v, Hq, Hkv, seqs)
    grads = ops.attn_packed_bwd(q, k, v, o, do, lse, Hq, Hkv, seqs)
    for name, t in zip(("o", "dq", "dk", "dv"), (o, *grads)):
        within(name, t, ref)
    assert all(torch.equal(a, b) for a, b in zip(grads, ops.attn_packed_bwd(q, k, v, o, do, lse, Hq, Hkv, seqs)))


# every sequence within one block of 32 rows on both sides (or with no rows at all)
SHORT = [
    ([1, 32, 20, 0, 7], None, True, 8, 2, 64),
    ([20, 32, 3], [32, 5, 30], True, 4, 1, 128),   # fewer keys than queries, and more
    ([31, 2, 17], [9, 32, 1], False, 6, 6, 128),
    ([18], [25], False, 16, 2, 64),
    ([0, 0], None, True, 2, 1, 64),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("case", range(len(SHORT)))
def test_short_sequences_match_float64(case, dtype):
    ops = _ops()
    lq, lk, causal, Hq, Hkv, dh = SHORT[case]
    q, k, v, do = _inputs(lq, lk or lq, Hq, Hkv, dh, dtype, 300 + case, extra=2)
    scale = 1 / math.sqrt(dh)
    ref = reference(q, k, v, do, lq, lk or lq, Hq, Hkv, causal, scale, E16 if dtype == torch.bfloat16 else 0.0)
    seqs = ops.PackedSeqs(lq, lk, causal=causal, device=DEV)
    assert seqs.c.one_block == 1
    o, lse = ops.attn_packed_fwd(q, k, v, Hq, Hkv, seqs)
    grads = ops.attn_packed_bwd(q, k, v, o, do, lse, Hq, Hkv, seqs)
    for name, t in zip(("o", "dq", "dk", "dv"), (o, *grads)):
        within(name, t, ref)
    assert all(torch.equal(a, b) for a, b in zip(grads, ops.attn_packed_bwd(q, k, v, o, do, lse, Hq, Hkv, seqs)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_packed_attention_matches_float64(case, dtype):
    ops = _ops()
    lq, lk, causal, Hq, Hkv, dh = CASES[case]
    q, k, v, do = _inputs(lq, lk or lq, Hq, Hkv, dh, dtype, 100 + case)
    scale = 1 / math.sqrt(dh)
    ref = reference(q, k, v, do, lq, lk or lq, Hq, Hkv, causal, scale, E16 if dtype == torch.bfloat16 else 0.0)
    seqs = ops.PackedSeqs(lq, lk, causal=causal, device=DEV)
    o, lse = ops.attn_packed_fwd(q, k, v, Hq, Hkv, seqs)
    assert o.dtype == dtype and lse.dtype == torch.float32
    within("o", o, ref)
    within("lse", lse, ref)
    dq, dk, dv = ops.attn_packed_bwd(q, k, v, o, do, lse, Hq, Hkv, seqs)
    within("dv", dv, ref)
    within("dq", dq, ref)
    within("dk", dk, ref)
    again = ops.attn_packed_bwd(q, k, v, o, do, lse, Hq, Hkv, seqs)
    assert all(torch.equal(a, b) for a, b in zip((dq, dk, dv), again))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lq", [[40, 7, 90], [300, 150, 260]], ids=["short", "tall"])
def test_rows_behind_the_last_sequence_and_columns_beside_stay(lq, dtype):
    ops = _ops()
    Hq, Hkv, dh, extra = 4, 2, 64, 37
    q, k, v, do = _inputs(lq, lq, Hq, Hkv, dh, dtype, 5, extra)
    n = sum(lq)
    for t in (q, k, v, do):
        t[n:] = float("nan")  # what lies there must not reach anything either
    seqs = ops.PackedSeqs(lq, device=DEV)
    blocks = [torch.full((n + extra, 3 * w), 7.0, dtype=dtype, device=DEV) for w in (Hq * dh, Hq * dh, Hkv * dh, Hkv * dh)]
    o, dq, dk, dv = (b[:, b.shape[1] // 3:2 * b.shape[1] // 3] for b in blocks)
    _, lse = ops.attn_packed_fwd(q, k, v, Hq, Hkv, seqs, out=o)
    ops.attn_packed_bwd(q, k, v, o, do, lse, Hq, Hkv, seqs, dq=dq, dk=dk, dv=dv)
    ref = reference(q[:n], k[:n], v[:n], do[:n], lq, lq, Hq, Hkv, True, 0.125, E16 if dtype == torch.bfloat16 else 0.0)
    for name, t, b in zip(("o", "dq", "dk", "dv"), (o, dq, dk, dv), blocks):
        within(name, t[:n], ref)
        w = b.shape[1] // 3
        assert bool((b[n:] == 7).all() and (b[:, :w] == 7).all() and (b[:, 2 * w:] == 7).all())
    new, lse2 = ops.attn_packed_fwd(q, k, v, Hq, Hkv, seqs)
    assert torch.equal(new[:n], o[:n]) and bool((new[n:] == 0).all()) and bool((lse2[:, n:] == 0).all())


@pytest.mark.gpu
def test_scale_raised_maxima_and_masked_extremes():
    """Scores that climb along the keys (the running maximum is raised again and again), a scale of the caller's, and keys of
    the type's lowest value in front of ordinary ones."""
    ops = _ops()
    lq, Hq, Hkv, dh, scale = [200, 70], 2, 1, 64, 0.3
    for dtype in (torch.bfloat16, torch.float32):
        q, k, v, do = _inputs(lq, lq, Hq, Hkv, dh, dtype, 9)
        k *= torch.linspace(0.1, 3, 270, device=DEV).to(dtype)[:, None]
        seqs = ops.PackedSeqs(lq, device=DEV)
        ref = reference(q, k, v, do, lq, lq, Hq, Hkv, True, scale, E16 if dtype == torch.bfloat16 else 0.0)
        o, lse = ops.attn_packed_fwd(q, k, v, Hq, Hkv, seqs, scale=scale)
        within("o", o, ref)
        within("lse", lse, ref)
        for n, t in zip(("dq", "dk", "dv"), ops.attn_packed_bwd(q, k, v, o, do, lse, Hq, Hkv, seqs, scale=scale)):
            within(n, t, ref)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_non_finite_rows_stay_in_their_sequence(dtype):
    ops = _ops()
    lq, Hq, Hkv, dh = [40, 50, 45, 200], 2, 2, 64
    q, k, v, do = _inputs(lq, lq, Hq, Hkv, dh, dtype, 21)
    seqs = ops.PackedSeqs(lq, device=DEV)
    clean, lse = ops.attn_packed_fwd(q, k, v, Hq, Hkv, seqs)
    grads = ops.attn_packed_bwd(q, k, v, clean, do, lse, Hq, Hkv, seqs)
    for t in (k, v, q, do):
        t[40:90] = float("nan")
        t[50] = float("inf")
    o, lse2 = ops.attn_packed_fwd(q, k, v, Hq, Hkv, seqs)
    got = ops.attn_packed_bwd(q, k, v, o, do, lse2, Hq, Hkv, seqs)
    for a, b in zip((o,) + tuple(got), (clean,) + tuple(grads)):
        assert torch.equal(a[:40], b[:40]) and torch.equal(a[90:], b[90:]) and bool(a[40:90].isnan().any())


@pytest.mark.gpu
def test_autograd_against_differences():
    """<grad, d> against the central difference of the fp32 forward along d = sign(grad), where the derivative stands out from
    the worst-case rounding of the values; the truncation of the difference is computed in float64."""
    from imagecaption_amd import functional
    ops = _ops()
    lq, lk, Hq, Hkv, dh, h = [30, 7, 140], [40, 7, 100], 4, 2, 64, 2.0 ** -5
    q, k, v, do = _inputs(lq, lk, Hq, Hkv, dh, torch.float32, 31)
    seqs = ops.PackedSeqs(lq, lk, device=DEV)
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
    functional.attn_packed(*leaves, Hq, Hkv, seqs).backward(do)
    ref = reference(q, k, v, do, lq, lk, Hq, Hkv, True, 0.125, 0.0)
    for i, name in enumerate(("dq", "dk", "dv")):
        d = ref[name][0].sign().float().to(DEV)
        side, exact, slack = [], [], 0.0
        for sign in (h, -h):
            args = [t + sign * d if j == i else t for j, t in enumerate((q, k, v))]
            o, _ = ops.attn_packed_fwd(*args, Hq, Hkv, seqs)
            r = reference(*args, do, lq, lk, Hq, Hkv, True, 0.125, 0.0)["o"]
            side.append(float((o.double() * do.double()).sum()))
            exact.append(float((r[0] * do.double().cpu()).sum()))
            slack += float((r[1] * do.double().cpu().abs()).sum())
        along = float((leaves[i].grad.double() * d.double()).sum())
        truncation = abs((exact[0] - exact[1]) / (2 * h) - float((ref[name][0] * d.double().cpu()).sum()))
        allowed = truncation + slack / (2 * h) + float((ref[name][1] * d.double().cpu().abs()).sum())
        assert abs((side[0] - side[1]) / (2 * h) - along) <= allowed
        assert allowed < 0.2 * (abs(along) + 1), (name, allowed, along)  # the check says something


@pytest.mark.gpu
def test_a_single_row_and_gradients_of_any_layout():
    """One packed row (whose row stride means nothing), gradients that arrive expanded or transposed, bf16 leaves."""
    from imagecaption_amd import functional
    ops = _ops()
    for lq in ([1], [3, 40]):
        q, k, v, do = _inputs(lq, lq, 2, 1, 64, torch.bfloat16, 61)
        seqs = ops.PackedSeqs(lq, device=DEV)
        o, lse = ops.attn_packed_fwd(q, k, v, 2, 1, seqs)
        for grad in (torch.ones_like(o), do):
            want = ops.attn_packed_bwd(q, k, v, o, grad.contiguous(), lse, 2, 1, seqs)
            leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
            got = functional.attn_packed(*leaves, 2, 1, seqs)
            assert torch.equal(got, o)
            if grad is do:
                got.backward(do.t().contiguous().t())
            else:
                got.sum().backward()
            assert all(torch.equal(a.grad, b) for a, b in zip(leaves, want))
            # a gradient that starts two bytes into its memory
            leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
            joined = torch.cat([o.new_zeros(1), functional.attn_packed(*leaves, 2, 1, seqs).flatten()])
            joined.backward(torch.cat([o.new_zeros(1), grad.flatten()]))
            assert all(torch.equal(a.grad, b) for a, b in zip(leaves, want))
        leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
        first = torch.autograd.grad(functional.attn_packed(*leaves, 2, 1, seqs), leaves, do.clone().requires_grad_(True), create_graph=True)
        with pytest.raises(RuntimeError):  # no second derivatives, and none that are silently zero
            torch.autograd.grad(sum(g.float().sum() for g in first), leaves)
        if lq == [1]:  # one key: the softmax is 1 whatever the score
            assert bool((want[0] == 0).all()) and bool((want[1] == 0).all()) and torch.equal(o[:, :64], v)
            turned = q.reshape(-1, 1).contiguous().t()
            assert turned.stride(0) == 1
            assert torch.equal(ops.attn_packed_fwd(turned, k, v, 2, 1, seqs)[0], o)


@pytest.mark.gpu
def test_extreme_scales():
    """Scores that all but vanish, and scores that leave one key of each row."""
    ops = _ops()
    lq, Hq, Hkv, dh = [130, 5], 2, 2, 64
    for scale in (2.0 ** -60, 1e-6, 8.0):
        for dtype in (torch.bfloat16, torch.float32):
            q, k, v, do = _inputs(lq, lq, Hq, Hkv, dh, dtype, 71)
            seqs = ops.PackedSeqs(lq, device=DEV)
            ref = reference(q, k, v, do, lq, lq, Hq, Hkv, True, scale, E16 if dtype == torch.bfloat16 else 0.0)
            o, lse = ops.attn_packed_fwd(q, k, v, Hq, Hkv, seqs, scale=scale)
            within("o", o, ref)
            within("lse", lse, ref)
            for n, t in zip(("dq", "dk", "dv"), ops.attn_packed_bwd(q, k, v, o, do, lse, Hq, Hkv, seqs, scale=scale)):
                within(n, t, ref)


@pytest.mark.gpu
def test_captured_calls_and_other_streams():
    ops = _ops()
    lq, Hq, Hkv, dh = [20, 150, 9], 4, 2, 64
    q, k, v, do = _inputs(lq, lq, Hq, Hkv, dh, torch.bfloat16, 41)
    seqs = ops.PackedSeqs(lq, device=DEV)
    o, lse = ops.attn_packed_fwd(q, k, v, Hq, Hkv, seqs)
    ops.attn_packed_bwd(q, k, v, o, do, lse, Hq, Hkv, seqs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go, glse = ops.attn_packed_fwd(q, k, v, Hq, Hkv, seqs)
        grads = ops.attn_packed_bwd(q, k, v, go, do, glse, Hq, Hkv, seqs)
    for turn in range(4):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(turn)))
        graph.replay()
        o, lse = ops.attn_packed_fwd(q, k, v, Hq, Hkv, seqs)
        eager = ops.attn_packed_bwd(q, k, v, o, do, lse, Hq, Hkv, seqs)
        torch.cuda.synchronize()
        assert torch.equal(o, go) and torch.equal(lse, glse) and all(torch.equal(a, b) for a, b in zip(eager, grads))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o2, lse2 = ops.attn_packed_fwd(q, k, v, Hq, Hkv, seqs)
        got = ops.attn_packed_bwd(q, k, v, o2, do, lse2, Hq, Hkv, seqs)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(o, o2) and all(torch.equal(a, b) for a, b in zip(eager, got))


@pytest.mark.gpu
@pytest.mark.parametrize("lq", [[20, 9, 32], [20, 150, 9]], ids=["short", "long"])
def test_a_captured_step_through_autograd(lq):
    """Forward and backward captured together and replayed with new contents.  No eager graph of the leaves is alive then."""
    from imagecaption_amd import functional
    ops = _ops()
    q, k, v, do = (t.contiguous() for t in _inputs(lq, lq, 4, 2, 64, torch.bfloat16, 91))
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    seqs = ops.PackedSeqs(lq, device=DEV)

    def step():
        for t in leaves:
            t.grad = None
        functional.attn_packed(*leaves, 4, 2, seqs).backward(do)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    for t in leaves:
        t.grad = None
    with torch.cuda.graph(graph):
        functional.attn_packed(*leaves, 4, 2, seqs).backward(do)
    for turn in range(4):
        with torch.no_grad():
            for i, t in enumerate(leaves):
                t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(10 * turn + i)))
        graph.replay()
        o, lse = ops.attn_packed_fwd(*(t.detach() for t in leaves), 4, 2, seqs)
        want = ops.attn_packed_bwd(*(t.detach() for t in leaves), o, do, lse, 4, 2, seqs)
        torch.cuda.synchronize()
        assert all(torch.equal(t.grad, w) for t, w in zip(leaves, want))


@pytest.mark.gpu
def test_a_plan_made_while_its_memory_is_still_written():
    """The allocator hands out blocks that work queued on the same stream may still write."""
    from imagecaption_amd._capi import CapdecError
    ops = _ops()
    lengths = [300 + i for i in range(200)]
    want = ops.PackedSeqs(lengths, device=DEV)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        block = torch.empty_like(want.table)
        at = block.data_ptr()
        torch.cuda._sleep(20_000_000)
        block.fill_(255)
        del block
        got = ops.PackedSeqs(lengths, device=DEV)
    side.synchronize()
    assert got.table.data_ptr() == at  # the test means something
    assert torch.equal(got.table, want.table)
    graph = torch.cuda.CUDAGraph()
    x = torch.zeros(4, device=DEV)
    with torch.cuda.graph(graph):
        x += 1
        with pytest.raises(CapdecError, match="before the capture"):
            ops.PackedSeqs([3], device=DEV)
    graph.replay()
    assert x.tolist() == [1.0] * 4


@pytest.mark.gpu
def test_a_plan_freed_while_another_stream_reads_it():
    ops = _ops()
    lq, Hq, Hkv, dh = [700] * 40, 4, 4, 64
    q, k, v, _ = _inputs(lq, lq, Hq, Hkv, dh, torch.bfloat16, 81)
    seqs = ops.PackedSeqs(lq, device=DEV)
    want, _ = ops.attn_packed_fwd(q, k, v, Hq, Hkv, seqs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    seqs = ops.PackedSeqs(lq, device=DEV)
    at, size = seqs.table.data_ptr(), seqs.table.numel()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        got, _ = ops.attn_packed_fwd(q, k, v, Hq, Hkv, seqs)
    del seqs
    later = torch.empty(size, dtype=torch.uint8, device=DEV)  # on the table's own stream: must not be its block yet
    assert later.data_ptr() != at
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_plans_and_arguments_are_refused_without_a_gpu():
    from imagecaption_amd import _capi
    from imagecaption_amd._capi import CapdecError
    ops = _ops()
    for bad in ([], [-1], [3, -2], [1 << 30, 1 << 30], [(1 << 31) - 1]):
        with pytest.raises(CapdecError):
            ops.PackedSeqs(bad, device=DEV)
    with pytest.raises(CapdecError):
        ops.PackedSeqs([3, 4], [3], device=DEV)
    with pytest.raises(CapdecError, match="no CPU fallback"):
        ops.PackedSeqs([3], device="cpu")
    lib = _capi.lib()
    ints = lambda *v: (C.c_int * len(v))(*v)
    assert lib.capdec_packed_table_bytes(ints(3, -1), None, 2) == 0
    assert lib.capdec_packed_table_bytes(ints((1 << 31) - 1), None, 1) == 0 and lib.capdec_packed_table_bytes(ints(1), ints((1 << 31) - 1024), 1) == 0
    assert lib.capdec_packed_table_bytes(ints(128, 0, 129), None, 3) == 32 * 2 * (1 + 2 + 2 + 3 + 4 + 5)
    s = _capi.PackedSeqs()
    assert lib.capdec_packed_plan(ints(3), None, 1, 1, 16, 1, C.byref(s)) == -4  # the table does not fit
    assert lib.capdec_packed_plan(ints(3), ints(-1), 1, 1, 16, 1024, C.byref(s)) == -1
    s.rows_q = s.rows_k = 3
    s.tiles[:] = [1] * 6
    s.table = 16
    good = dict(q=16, ldq=128, k=16, ldk=64, v=16, ldv=64, o=16, ldo=128, Hq=2, Hkv=1, dh=64, dtype=0, scale=0.1, rows=3)
    for change in (dict(Hq=3, Hkv=2), dict(Hkv=0), dict(dh=32), dict(dtype=1), dict(scale=0.0), dict(scale=-1.0),
                   dict(scale=math.inf), dict(scale=1e-30), dict(q=None), dict(k=8), dict(ldq=126), dict(ldk=65), dict(ldo=64), dict(rows=2)):
        a = dict(good, **change)
        assert lib.capdec_attn_packed_fwd(C.byref(s), a["q"], a["ldq"], a["k"], a["ldk"], a["v"], a["ldv"], a["o"], a["ldo"], 16,
                                          a["rows"], a["Hq"], a["Hkv"], a["dh"], a["dtype"], a["scale"], None) == -1, change
        assert lib.capdec_last_error()
    assert lib.capdec_attn_packed_bwd(C.byref(s), 16, 128, 16, 64, 16, 64, 16, 128, 16, 128, None, 3, 16, 1 << 20, 16, 128, 16, 64, 16, 64,
                                      2, 1, 64, 0, 0.1, None) == -1  # no lse
    need = lib.capdec_attn_packed_scratch_bytes(C.byref(s), 3, 2, 1, 64, 3)
    assert need >= 2 * 3 * 16
    for scratch, size, rc in ((None, need, -1), (8, need, -1), (16, need - 1, -4)):
        assert lib.capdec_attn_packed_bwd(C.byref(s), 16, 128, 16, 64, 16, 64, 16, 128, 16, 128, 16, 3, scratch, size, 16, 128, 16, 64,
                                          16, 64, 2, 1, 64, 3, 0.1, None) == rc


@pytest.mark.gpu
def test_tensors_that_do_not_fit_are_refused():
    from imagecaption_amd._capi import CapdecError
    ops = _ops()
    lq, Hq, Hkv, dh = [5, 9], 4, 2, 64
    q, k, v, do = _inputs(lq, lq, Hq, Hkv, dh, torch.bfloat16, 51)
    seqs = ops.PackedSeqs(lq, device=DEV)
    o, lse = ops.attn_packed_fwd(q, k, v, Hq, Hkv, seqs)
    odd = torch.zeros(14, Hq * dh + 3, dtype=torch.bfloat16, device=DEV)
    for args in ((q.float(), k, v), (q.half(), k.half(), v.half()), (q[:13], k, v), (q, k[:, :64], v), (odd[:, :Hq * dh], k, v),
                 (odd[:, 3:], k, v), (q.t(), k, v), (q.cpu(), k, v)):
        with pytest.raises(CapdecError):
            ops.attn_packed_fwd(*args, Hq, Hkv, seqs)
    for heads in ((3, 2), (4, 0), (8, 2), (2, 2)):
        with pytest.raises(CapdecError):
            ops.attn_packed_fwd(q, k, v, *heads, seqs)
    for bad in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(CapdecError):
            ops.attn_packed_fwd(q, k, v, Hq, Hkv, seqs, scale=bad)
    with pytest.raises(CapdecError):
        ops.attn_packed_bwd(q, k, v, o, do, lse.t(), Hq, Hkv, seqs)
    wide = torch.empty((1 << 32) + 512, dtype=torch.bfloat16, device=DEV)
    two = ops.PackedSeqs([2], device=DEV)
    for far in ((1 << 32) + 256, 1 << 25):  # a row stride that 32 bits would cut to 256; one of more than 2^25 bytes
        with pytest.raises(CapdecError):
            ops.attn_packed_fwd(wide.as_strided((2, Hq * dh), (far, 1)), k, v, Hq, Hkv, two)
    with pytest.raises(CapdecError):
        ops.attn_packed_bwd(q, k, v, o, do, lse, Hq, Hkv, seqs, dk=torch.zeros(14, 64, dtype=torch.bfloat16, device=DEV))


@pytest.mark.gpu
def test_an_argument_without_a_truth_value_is_its_own_error():
    import numpy as np
    ops = _ops()
    q, k, v, _ = (t.contiguous() for t in _inputs([5, 9], [5, 9], 4, 2, 64, torch.bfloat16, 51))
    seqs = ops.PackedSeqs([5, 9], device=DEV)
    ops.attn_packed_fwd(q, k, v, 4, 2, seqs)
    with pytest.raises(ValueError, match="truth value"):
        ops.attn_packed_fwd(q, k, v, 4, 2, seqs, save_lse=np.array([1, 0]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lq", [[20, 9, 32], [300, 70]], ids=["short", "long"])
def test_scores_up_to_the_documented_size_stay_finite(lq, dtype):
    """Scaled scores of up to 2^24: weights say little there, but no row becomes NaN or one that sees nothing."""
    ops = _ops()
    q, k, v, do = _inputs(lq, lq, 4, 2, 64, dtype, 95)
    top = max(float((a.float() @ b.float().T).abs().max()) for a in q.split(64, 1) for b in k.split(64, 1))
    scale = 2.0 ** 24 / top
    seqs = ops.PackedSeqs(lq, device=DEV)
    o, lse = ops.attn_packed_fwd(q, k, v, 4, 2, seqs, scale=scale)
    assert float(lse.abs().max()) > 2.0 ** 20  # the test means something
    for t in (o, lse, *ops.attn_packed_bwd(q, k, v, o, do, lse, 4, 2, seqs, scale=scale)):
        assert bool(t.isfinite().all())
