"""Workloads of the serving / ragged-training operators, with their plain forms.

Four operators, in the order a program that trains on captions of different lengths and then serves them uses them:

* ``packed``  -- attention over sequences of different lengths packed into one block of rows, grouped heads, causal
                 or not; ``train`` adds the gradients;
* ``cache``   -- new key / value rows written into a paged cache (rounded to e4m3 with one scale for each token and
                 head, or kept as bf16), and read back as rows;
* ``paged``   -- attention of a chunk of new tokens (one or more for each sequence) over that paged cache;
* ``verify``  -- drafted tokens accepted or replaced against the target model's probabilities, from given uniforms.

``run`` computes them in elementary torch operations while ``own`` is false, and calls the package while it is true.
"""
import math
import random

import numpy as np
import torch

own = False
DEV = "cuda"
E4M3_MAX = 448.0
AMAX_FLOOR = 2.0 ** -100


# ---- the cases --------------------------------------------------------------------------------------------------------
def listed():
    return [
        # C2 of this framework's benchmark (256 captions of 8 .. 20 tokens, 8 heads of 64), without its padding
        dict(name="captions train bf16", op="packed", train=True, dtype="bf16", n=256, low=8, high=20, mem=0, hq=8, hkv=8,
             dh=64, salt=1),
        # C1: the reference's own paragraph captions, up to 299 tokens, in its own precision
        dict(name="paragraphs train fp32", op="packed", train=True, dtype="fp32", n=32, low=40, high=299, mem=0, hq=8, hkv=8,
             dh=64, salt=2),
        # a ragged training batch of long texts, grouped heads
        dict(name="long texts train bf16", op="packed", train=True, dtype="bf16", n=8, low=300, high=4096, mem=0, hq=16,
             hkv=4, dh=128, salt=3),
        # prompts of one prefill step, the longest several thousand tokens
        dict(name="prompts bf16", op="packed", train=False, dtype="bf16", n=6, low=37, high=6144, mem=0, hq=16, hkv=2,
             dh=128, salt=4),
        # one decode step of a few captions: a handful of short contexts, where the launch counts
        dict(name="decode small bf16", op="paged", dtype="bf16", n=4, low=1, high=299, qlow=1, qhigh=1, hq=8, hkv=8, dh=64,
             page=16, salt=5),
        # one decode step of a few long conversations: 60 thousand cached tokens each at most
        dict(name="decode long e4m3", op="paged", dtype="e4m3", n=8, low=9000, high=60001, qlow=1, qhigh=1, hq=32, hkv=4,
             dh=128, page=64, salt=6),
        # five tokens a sequence: four drafted ones and the one before them
        dict(name="draft chunk e4m3", op="paged", dtype="e4m3", n=48, low=100, high=8000, qlow=2, qhigh=5, hq=16, hkv=4,
             dh=128, page=16, salt=7),
        # chunked prefill: several hundred new tokens over what is cached already
        dict(name="prefill chunk bf16", op="paged", dtype="bf16", n=4, low=1500, high=8192, qlow=200, qhigh=511, hq=16,
             hkv=4, dh=128, page=32, salt=8),
        # the cache rows of one decode step
        dict(name="cache step e4m3", op="cache", dtype="e4m3", rows=64, hkv=4, dh=128, page=16, salt=9),
        # the cache rows of a prefill
        dict(name="cache prefill e4m3", op="cache", dtype="e4m3", rows=40001, hkv=8, dh=128, page=32, salt=10),
        # a few captions over this framework's C2 vocabulary
        dict(name="verify small", op="verify", n=3, drafts=3, vocab=10000, salt=11),
        # a full serving batch over the C3 vocabulary
        dict(name="verify batch", op="verify", n=256, drafts=7, vocab=30000, salt=12),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["packed", "packed", "train", "train", "paged", "paged", "paged", "cache", "verify"])
    hkv, group, dh = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 1, 2, 4, 5, 8]), rng.choice([64, 128])
    salt = rng.randrange(1000, 1000000)
    if op in ("packed", "train"):
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
        high = _log_int(rng, 1, 4096 if dtype == "bf16" else 1000)
        # the plain form's score block (padded) stays under 1.2e9 elements
        n = _log_int(rng, 1, max(1, min(256, int((1.2e9 if dtype == "bf16" else 2e8) / (hkv * group * high * high)))))
        mem = rng.choice([0, 0, 0, rng.randrange(1, 260)])  # > 0: not causal, over a memory of that many rows at most
        return dict(op="packed", train=op == "train", dtype=dtype, n=n, low=max(1, high // rng.choice([1, 3, 20])), high=high,
                    mem=mem, hq=hkv * group, hkv=hkv, dh=dh, salt=salt)
    if op == "paged":
        qhigh = rng.choice([1, 1, 1, 2, 5, 9, 64, 200])
        high = _log_int(rng, max(qhigh, 8), 30000 if qhigh < 10 else 6000)
        n = _log_int(rng, 1, max(1, min(128, int(min(1.2e8 / (hkv * dh * high), 1e9 / (hkv * group * qhigh * high))))))
        return dict(op="paged", dtype=rng.choice(["bf16", "e4m3"]), n=n, low=max(1, high // rng.choice([1, 5, 50])), high=high,
                    qlow=rng.randrange(1, qhigh + 1), qhigh=qhigh, hq=hkv * group, hkv=hkv, dh=dh,
                    page=rng.choice([8, 16, 32, 64, 128]), salt=salt)
    if op == "cache":
        return dict(op="cache", dtype=rng.choice(["bf16", "e4m3", "e4m3"]), rows=_log_int(rng, 1, 30000), hkv=hkv, dh=dh,
                    page=rng.choice([8, 16, 32, 64, 128]), salt=salt)
    return dict(op="verify", n=_log_int(rng, 1, 200), drafts=rng.randrange(1, 9), vocab=_log_int(rng, 50, 33000), salt=salt)


def _lengths(n, low, high, salt):
    """n lengths, spread over the logarithm of low .. high, the longest among them."""
    rng = random.Random(salt)
    out = [_log_int(rng, low, high) for _ in range(n)]
    out[rng.randrange(n)] = high
    return out


def _packed_lengths(case):
    lq = _lengths(case["n"], case["low"], case["high"], case["salt"])
    return lq, (_lengths(case["n"], max(1, case["mem"] // 2), case["mem"], case["salt"] + 1) if case["mem"] else lq)


def _paged_lengths(case):
    new = _lengths(case["n"], case["qlow"], case["qhigh"], case["salt"] + 1)
    total = [max(a, b) for a, b in zip(_lengths(case["n"], case["low"], case["high"], case["salt"]), new)]
    return new, total


def _drafted(case):
    rng = random.Random(case["salt"])
    return [case["drafts"] if rng.random() < 0.7 else rng.randrange(0, case["drafts"] + 1) for _ in range(case["n"])]


def _pairs(lq, lk, causal):
    """How many (query, key) pairs are visible; a causal query i of nq sees the keys up to i + nk - nq."""
    if not causal:
        return sum(a * b for a, b in zip(lq, lk))
    return sum(a * (b - a) + a * (a + 1) // 2 for a, b in zip(lq, lk))  # nk >= nq in every case here


def work(case):
    if case["op"] == "packed":
        lq, lk = _packed_lengths(case)
        es = 2 if case["dtype"] == "bf16" else 4
        q, kv = sum(lq) * case["hq"] * case["dh"] * es, sum(lk) * case["hkv"] * case["dh"] * es
        flops = _pairs(lq, lk, not case["mem"]) * case["hq"] * case["dh"] * (14 if case["train"] else 4)
        stats = 4 * sum(lq) * case["hq"]
        # forward: q, k, v read, o and the row statistics written; training: the output's gradient read and dq, dk, dv written too
        return {"bytes": 2 * q + 2 * kv + stats + ((2 * q + 2 * kv) if case["train"] else 0), "flops": flops}
    if case["op"] == "paged":
        new, total = _paged_lengths(case)
        row = case["dh"] * 2 if case["dtype"] == "bf16" else case["dh"] + 4
        return {"bytes": 2 * sum(total) * case["hkv"] * row + 2 * 2 * sum(new) * case["hq"] * case["dh"],
                "flops": 4 * _pairs(new, total, True) * case["hq"] * case["dh"]}
    if case["op"] == "cache":
        rows = case["rows"] * case["hkv"]
        row = case["dh"] * 2 if case["dtype"] == "bf16" else case["dh"] + 4
        # write: bf16 rows in, cache rows out; read back: cache rows in, bf16 rows out; keys and values
        return {"bytes": 2 * rows * (2 * case["dh"] * 2 + 2 * row), "flops": 2 * rows * case["dh"] * 4}
    # one row of the target's and one of the draft's probabilities for each sequence, and the drafted tokens' entries
    return {"bytes": case["n"] * (8 * case["vocab"] + 24 * case["drafts"] + 16), "flops": case["n"] * case["vocab"] * 3}


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _starts(lengths):
    return [0] + np.cumsum(lengths).tolist()


def _pad_index(lengths):
    """[n, longest] row of the packed block for each place of the padded one (0 where there is none), and which there are."""
    pos = np.arange(max(lengths))
    there = pos[None, :] < np.asarray(lengths)[:, None]
    at = np.where(there, np.asarray(_starts(lengths)[:-1])[:, None] + pos[None, :], 0)
    return torch.from_numpy(at).to(DEV), torch.from_numpy(there).to(DEV)


def _quantised(x):
    """e4m3 codes and scales of rows [..., dh]."""
    scale = x.float().abs().amax(-1).clamp(min=AMAX_FLOOR) / E4M3_MAX
    return (x.float() / scale[..., None]).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    st = dict(case)
    if case["op"] == "packed":
        lq, lk = _packed_lengths(case)
        dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        hq, hkv, dh = case["hq"], case["hkv"], case["dh"]
        # queries, keys and values as a projection leaves them: column slices of one block where the lengths agree
        if case["mem"]:
            st["q"] = normal(sum(lq), hq * dh).to(dt)
            kv = normal(sum(lk), 2 * hkv * dh).to(dt)
        else:
            qkv = normal(sum(lq), (hq + 2 * hkv) * dh).to(dt)
            st["q"], kv = qkv[:, :hq * dh], qkv[:, hq * dh:]
        st["k"], st["v"] = kv[:, :hkv * dh], kv[:, hkv * dh:]
        if case["train"]:
            st["do"] = normal(sum(lq), hq * dh).to(dt)
        st["pad_q"], st["pad_k"] = _pad_index(lq), _pad_index(lk)
        if own:
            from imagecaption_amd import ops
            st["seqs"] = ops.PackedSeqs(lq, lk, causal=not case["mem"], device=DEV)
    elif case["op"] == "paged":
        new, total = _paged_lengths(case)
        ps, hkv, dh = case["page"], case["hkv"], case["dh"]
        need = [-(-t // ps) for t in total]
        pages = sum(need) + 3
        order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)  # pages come in no order
        at, there = _pad_index(need)
        st["table"] = torch.where(there, order[at], torch.zeros_like(order[at])).contiguous()
        k, v = normal(pages, hkv, ps, dh), normal(pages, hkv, ps, dh)
        if case["dtype"] == "e4m3":
            (st["k"], st["ks"]), (st["v"], st["vs"]) = _quantised(k), _quantised(v)
        else:
            st["k"], st["v"], st["ks"], st["vs"] = k.to(torch.bfloat16), v.to(torch.bfloat16), None, None
        st["q"] = normal(sum(new), case["hq"] * dh).to(torch.bfloat16)
        st["lens"] = torch.tensor(total, dtype=torch.int32, device=DEV)
        st["cu"] = torch.tensor(_starts(new), dtype=torch.int32, device=DEV)
        st["pad_q"], st["max_q"] = _pad_index(new), max(new)
    elif case["op"] == "cache":
        ps, hkv, dh = case["page"], case["hkv"], case["dh"]
        pages = -(-case["rows"] // ps) + 2
        kv = normal(case["rows"], 2 * hkv * dh).to(torch.bfloat16)
        # some channels of keys are far larger than the others
        kv[:, :hkv * dh] *= 1 + 15 * (torch.rand(hkv * dh, generator=g, device=DEV) < 0.05)
        st["k_new"], st["v_new"] = kv[:, :hkv * dh], kv[:, hkv * dh:]
        order = torch.randperm(pages, generator=g, device=DEV)
        r = torch.arange(case["rows"], device=DEV)
        st["slots"] = (order[r // ps] * ps + r % ps).to(torch.int32)
        dt = torch.float8_e4m3fn if case["dtype"] == "e4m3" else torch.bfloat16
        for x in "kv":
            st[x] = torch.zeros(pages, hkv, ps, dh, device=DEV).to(dt)
            st[x + "s"] = torch.zeros(pages, hkv, ps, device=DEV) if case["dtype"] == "e4m3" else None
    else:
        n, d, V = case["n"], case["drafts"], case["vocab"]
        logits = 2.5 * normal(n, d + 1, V)
        near = logits[:, :d] + 0.6 * normal(n, d, V)
        st["target"], st["draft"] = torch.softmax(logits, -1), torch.softmax(near, -1)
        noise = torch.rand(n, d, V, generator=g, device=DEV).clamp_(min=1e-20).log_().neg_()
        st["tokens"] = (st["draft"] / noise).argmax(-1)  # a draw from the draft's probabilities
        st["drafted"] = torch.tensor(_drafted(case), dtype=torch.int32, device=DEV)
        st["u_accept"], st["u_sample"] = torch.rand(n, d, generator=g, device=DEV), torch.rand(n, generator=g, device=DEV)
    if own and case["op"] in ("paged", "cache"):
        from imagecaption_amd import ops
        st["cache"] = ops.PagedKVCache(st["k"], st["v"], st["ks"], st["vs"])
    return st


# ---- one pass ---------------------------------------------------------------------------------------------------------
def run(st):
    return {"packed": _packed, "paged": _paged, "cache": _cache, "verify": _verify}[st["op"]](st)


def _heads(rows, at, heads):
    """[rows, heads * dh] -> fp32 [n, heads, longest, dh] of the padded block."""
    return rows.float()[at].unflatten(-1, (heads, -1)).transpose(1, 2)


def _packed(st):
    hq, hkv = st["hq"], st["hkv"]
    if own:
        from imagecaption_amd import ops
        o, lse = ops.attn_packed_fwd(st["q"], st["k"], st["v"], hq, hkv, st["seqs"])
        if not st["train"]:
            return {"o": o, "lse": lse}
        dq, dk, dv = ops.attn_packed_bwd(st["q"], st["k"], st["v"], o, st["do"], lse, hq, hkv, st["seqs"])
        return {"o": o, "dq": dq, "dk": dk, "dv": dv}
    (aq, tq), (ak, tk) = st["pad_q"], st["pad_k"]
    group, scale, dt = hq // hkv, 1.0 / math.sqrt(st["dh"]), st["q"].dtype
    q = _heads(st["q"], aq, hq)
    k = _heads(st["k"], ak, hkv).repeat_interleave(group, 1)
    v = _heads(st["v"], ak, hkv).repeat_interleave(group, 1)
    seen = tk[:, None, None, :].expand(-1, 1, aq.shape[1], -1)
    if not st["mem"]:
        i = torch.arange(aq.shape[1], device=DEV)
        seen = seen & (i[None, :] <= i[:, None])
    s = (q @ k.transpose(2, 3).contiguous()).mul_(scale).masked_fill_(~seen, float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = s.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(total)
    o = p @ v

    def rows(x, there, like):
        return x.transpose(1, 2).flatten(2)[there].to(like)

    out = {"o": rows(o, tq, dt)}
    if not st["train"]:
        out["lse"] = (m + total.log()).squeeze(-1).transpose(1, 2)[tq].t().contiguous()
        return out
    do = _heads(st["do"], aq, hq) * tq[:, None, :, None]
    dv = p.transpose(2, 3).contiguous() @ do
    ds = do @ v.transpose(2, 3).contiguous()
    ds = ds.sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dk = ds.transpose(2, 3).contiguous() @ q
    out["dq"] = rows(ds @ k, tq, dt)
    out["dk"] = rows(dk.unflatten(1, (hkv, group)).sum(2), tk, dt)
    out["dv"] = rows(dv.unflatten(1, (hkv, group)).sum(2), tk, dt)
    return out


def _paged(st):
    if own:
        from imagecaption_amd import ops
        cu = None if st["max_q"] == 1 else st["cu"]  # one new token for each sequence: row i is sequence i's
        return ops.attn_paged(st["q"], st["cache"], st["table"], st["lens"], st["hq"], cu_q=cu, max_q=st["max_q"])
    table, (aq, tq), hq, hkv = st["table"].long(), st["pad_q"], st["hq"], st["hkv"]

    def gathered(x, scale):
        x = x[table].float() if scale is None else x.view(torch.uint8)[table].view(x.dtype).float() * scale[table][..., None]
        return x.transpose(1, 2).flatten(2, 3)  # [n, hkv, keys, dh]

    group, longest = hq // hkv, aq.shape[1]
    q = _heads(st["q"], aq, hq).unflatten(1, (hkv, group)).flatten(2, 3)  # [n, hkv, group * longest, dh]
    k, v = gathered(st["k"], st["ks"]), gathered(st["v"], st["vs"])
    s = q @ k.transpose(2, 3).contiguous() / math.sqrt(st["dh"])
    lens, new = st["lens"].long(), tq.sum(1)
    last = (lens - new)[:, None] + torch.arange(longest, device=DEV)  # the last position that a row sees
    seen = (torch.arange(k.shape[2], device=DEV) <= last[..., None]) & tq[..., None]
    s = s.unflatten(2, (group, longest)).masked_fill_(~seen[:, None, None], float("-inf"))
    p = (s - s.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = (p.flatten(2, 3) @ v.masked_fill(torch.arange(v.shape[2], device=DEV)[:, None] >= lens[:, None, None, None], 0.0))
    return o.unflatten(2, (group, longest)).flatten(1, 2).transpose(1, 2).flatten(2)[tq].to(torch.bfloat16)


def _cache(st):
    hkv, dh, ps = st["hkv"], st["dh"], st["page"]
    if own:
        from imagecaption_amd import ops
        ops.kv_cache_write(st["cache"], st["k_new"], st["v_new"], st["slots"])
        k, v = ops.kv_cache_read(st["cache"], st["slots"])
        return {"k": k, "v": v, "pages_k": st["k"], "pages_v": st["v"], "scale_k": st["ks"], "scale_v": st["vs"]}
    page, row = st["slots"].long() // ps, st["slots"].long() % ps

    def both(pages, scales, new):
        new = new.unflatten(1, (hkv, dh))
        if scales is None:
            pages[page, :, row] = new
            return pages[page, :, row].flatten(1)
        codes, scale = _quantised(new)
        raw = pages.view(torch.uint8)
        raw[page, :, row], scales[page, :, row] = codes.view(torch.uint8), scale
        back = raw[page, :, row].view(pages.dtype).float() * scales[page, :, row][..., None]
        return back.to(torch.bfloat16).flatten(1)

    return {"k": both(st["k"], st["ks"], st["k_new"]), "v": both(st["v"], st["vs"], st["v_new"]), "pages_k": st["k"],
            "pages_v": st["v"], "scale_k": st["ks"], "scale_v": st["vs"]}


def _verify(st):
    if own:
        from imagecaption_amd import ops
        return ops.draft_verify(st["target"], st["draft"], st["tokens"], st["u_accept"], st["u_sample"],
                                num_draft=st["drafted"])
    target, draft, tokens, drafted = st["target"], st["draft"], st["tokens"], st["drafted"].long()
    n, d, V = draft.shape
    p = target[:, :d].gather(2, tokens[..., None]).squeeze(2).double()
    q = draft.gather(2, tokens[..., None]).squeeze(2).double()
    j = torch.arange(d + 1, device=DEV)
    taken = (st["u_accept"].double() * q < p) & (j[:d] < drafted[:, None])
    count = taken.long().cumprod(1).sum(1)
    b = torch.arange(n, device=DEV)
    whole = target[b, count].double()
    less = torch.where((count < drafted)[:, None], draft[b, count.clamp(max=d - 1)].double(), 0.0)
    w = (whole - less).clamp(min=0)
    w = torch.where(w.sum(1, keepdim=True) > 0, w, whole)
    sums = w.cumsum(1)
    pick = (sums <= st["u_sample"].double()[:, None] * sums[:, -1:]).sum(1)
    last = (w > 0).long().mul(torch.arange(V, device=DEV)).amax(1)
    new = torch.minimum(pick, last)
    padded = torch.cat([tokens, torch.zeros_like(tokens[:, :1])], 1)
    out = torch.where(j < count[:, None], padded, torch.where(j == count[:, None], new[:, None], 0))
    return out, count.to(torch.int32)


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    return {"packed": _exact_packed, "paged": _exact_paged, "cache": _exact_cache, "verify": _exact_verify}[case["op"]](case, st)


def _one(q, k, v, first):
    """Probabilities, output and log-sum-exp of one head of one sequence; row i sees the keys up to first + i."""
    s = (q @ k.t()) * q.shape[1] ** -0.5
    if first is not None:
        s = s + torch.full_like(s, -math.inf).triu(first + 1)
    lse = torch.logsumexp(s, 1)
    p = torch.exp(s - lse[:, None])
    return p, p @ v, lse


def _exact_packed(case, st):
    lq, lk = _packed_lengths(case)
    sq, sk, dh, group = _starts(lq), _starts(lk), case["dh"], case["hq"] // case["hkv"]
    x = {n: st[n].double() for n in ("q", "k", "v", "do") if n in st}
    out = {n: torch.zeros_like(x[m]) for n, m in (("o", "q"), ("dq", "q"), ("dk", "k"), ("dv", "v"))}
    lse = torch.zeros(case["hq"], sum(lq), dtype=torch.float64, device=DEV)
    for i in range(case["n"]):
        a, b = slice(sq[i], sq[i + 1]), slice(sk[i], sk[i + 1])
        for h in range(case["hq"]):
            c, e = slice(h * dh, (h + 1) * dh), slice(h // group * dh, (h // group + 1) * dh)
            q, k, v = x["q"][a, c], x["k"][b, e], x["v"][b, e]
            p, o, lse[h, a] = _one(q, k, v, None if case["mem"] else 0)
            out["o"][a, c] = o
            if case["train"]:
                do = x["do"][a, c]
                dp = do @ v.t()
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) * dh ** -0.5
                out["dq"][a, c] = ds @ k
                out["dk"][b, e] += ds.t() @ q
                out["dv"][b, e] += p.t() @ do
    return out if case["train"] else {"o": out["o"], "lse": lse}


def _exact_paged(case, st):
    new, total = _paged_lengths(case)
    at, dh, group, ps = _starts(new), case["dh"], case["hq"] // case["hkv"], case["page"]
    out = torch.zeros(sum(new), case["hq"] * dh, dtype=torch.float64, device=DEV)
    for i, (a, t) in enumerate(zip(new, total)):
        pages = st["table"][i, :-(-t // ps)].long()
        for h in range(case["hkv"]):
            k, v = ((st[x].view(torch.uint8)[pages, h].view(st[x].dtype) if st[x + "s"] is not None else st[x][pages, h]).double()
                    for x in "kv")
            if st["ks"] is not None:
                k, v = k * st["ks"][pages, h].double()[..., None], v * st["vs"][pages, h].double()[..., None]
            k, v = k.flatten(0, 1)[:t], v.flatten(0, 1)[:t]
            for j in range(h * group, (h + 1) * group):
                c = slice(j * dh, (j + 1) * dh)
                out[at[i]:at[i + 1], c] = _one(st["q"][at[i]:at[i + 1], c].double(), k, v, t - a)[1]
    return out


def _exact_cache(case, st):
    slots = st["slots"].long()
    pages, hkv, ps, dh = st["k"].shape
    out = {}
    for x in "kv":
        rows = st[x + "_new"].double().reshape(-1, hkv, dh)
        held, scale = rows, None
        if st[x + "s"] is not None:
            scale = rows.abs().max(-1).values / E4M3_MAX
            # e4m3: three mantissa bits, the smallest step 2^-9; the nearest value, ties to the even one
            y = rows / scale[..., None]
            step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
            held = torch.round(y / step) * step
        flat = torch.zeros(pages * ps, hkv, dh, dtype=torch.float64, device=DEV)
        flat[slots] = held
        out["pages_" + x] = flat.view(pages, ps, hkv, dh).transpose(1, 2).contiguous()
        out["scale_" + x] = None
        if scale is not None:
            flat = torch.zeros(pages * ps, hkv, dtype=torch.float64, device=DEV)
            flat[slots] = scale
            out["scale_" + x] = flat.view(pages, ps, hkv).transpose(1, 2).contiguous()
            held = held * scale[..., None]
        out[x] = held.reshape(-1, hkv * dh)
    return out


def _exact_verify(case, st):
    # row by row on the host, in double
    u, us, tok = st["u_accept"].cpu().numpy(), st["u_sample"].cpu().numpy(), st["tokens"].cpu().numpy()
    out, counts = np.zeros((case["n"], case["drafts"] + 1), np.int64), np.zeros(case["n"], np.int32)
    for b, drafted in enumerate(_drafted(case)):
        target, draft = (st[x][b].cpu().numpy().astype(np.float64) for x in ("target", "draft"))
        i = 0
        while i < drafted and float(u[b, i]) * draft[i, tok[b, i]] < target[i, tok[b, i]]:
            out[b, i] = tok[b, i]
            i += 1
        w = np.maximum(target[i] - draft[i], 0) if i < drafted else target[i]
        w = target[i] if w.sum() <= 0 else w
        sums = np.cumsum(w)
        out[b, i] = min(np.searchsorted(sums, float(us[b]) * sums[-1], side="right"), np.nonzero(w)[0][-1])
        counts[b] = i
    return torch.from_numpy(out), torch.from_numpy(counts)
