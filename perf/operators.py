"""Performance cases of the operators that a model's serving and training need around plain attention.

Three operators: attention whose scores are capped, biased by distance or
masked by document and prefix (prefill, training step, single-token decode);
a paged cache held in 8 bits with a scale for each page and head (the append
that writes it, the decode that reads it); and eviction from a cache by
accumulated attention weight (the decode that accumulates it, the compaction).

``own`` chooses what ``run`` does: False computes the operators in elementary
torch operations in 32 bits, True calls the module.  ``listed()`` are fixed
cases, ``draw()`` gives others of the same ranges, ``exact()`` is the operators'
definition in 64 bits.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

HALF = torch.float16
E4M3 = torch.float8_e4m3fn
CODE_MAX = {"int8": 127.0, "e4m3": 448.0}


def listed():
    return [
        # a fine-tuning step of a small model with capped scores: launch and latency bound
        {"name": "train_capped_small", "kind": "train", "dtype": "float16", "B": 1, "HQ": 8, "HKV": 8, "N": 256,
         "D": 64, "causal": True, "cap": 50.0, "bias": False, "docs": 0, "prefix": 0, "mix": 0},
        # one layer of a pretraining step: packed documents, grouped KV heads, capped scores; the largest step
        {"name": "train_capped_docs", "kind": "train", "dtype": "float16", "B": 4, "HQ": 32, "HKV": 8, "N": 2048,
         "D": 128, "causal": True, "cap": 50.0, "bias": False, "docs": 600, "prefix": 0, "mix": 1},
        # single precision, a ragged length, distance bias and a prefix that all rows see
        {"name": "train_bias_prefix_fp32", "kind": "train", "dtype": "float32", "B": 2, "HQ": 16, "HKV": 16,
         "N": 1000, "D": 64, "causal": True, "cap": 0.0, "bias": True, "docs": 0, "prefix": 250, "mix": 2},
        # one long prompt with capped scores: the largest prefill
        {"name": "prefill_capped_long", "kind": "prefill", "B": 1, "HQ": 32, "HKV": 8, "N": 8192, "D": 128,
         "causal": True, "cap": 50.0, "bias": False, "docs": 0, "prefix": 0, "mix": 3},
        # padded sequences through a bidirectional tower with a distance bias, 80-wide heads
        {"name": "prefill_bias_d80", "kind": "prefill", "B": 8, "HQ": 16, "HKV": 16, "N": 577, "D": 80,
         "causal": False, "cap": 0.0, "bias": True, "docs": 400, "prefix": 0, "mix": 4},
        # interactive decode of one sequence with capped scores
        {"name": "decode_capped_single", "kind": "decode", "B": 1, "HQ": 32, "HKV": 8, "N": 4097, "D": 128, "lo": 16,
         "cap": 50.0, "bias": False, "mix": 5},
        # a server's decode step over ragged sequences with a distance bias
        {"name": "decode_bias_batch", "kind": "decode", "B": 64, "HQ": 32, "HKV": 8, "N": 8193, "D": 128, "lo": 16,
         "cap": 0.0, "bias": True, "mix": 6},
        # a few sequences' step on an 8-bit cache: append the token, attend
        {"name": "kv8_step_small", "kind": "kv8_step", "codes": "int8", "B": 4, "HQ": 32, "HKV": 8, "hi": 1024,
         "D": 128, "lo": 64, "page": 16, "cap": 0.0, "mix": 7},
        # a full server's step on an 8-bit cache with scattered pages
        {"name": "kv8_step_batch", "kind": "kv8_step", "codes": "e4m3", "B": 128, "HQ": 32, "HKV": 8, "hi": 4096,
         "D": 128, "lo": 64, "page": 16, "cap": 0.0, "mix": 8},
        # prompts of mixed lengths written to the 8-bit cache after their prefill
        {"name": "kv8_prompts", "kind": "kv8_prompts", "codes": "int8", "B": 16, "HKV": 8, "lo": 128, "hi": 2048,
         "D": 128, "page": 16, "mix": 9},
        # a decode step that adds up what each cached token was attended with
        {"name": "weighted_decode", "kind": "weighted", "B": 16, "HQ": 32, "HKV": 8, "N": 4096, "D": 128, "lo": 512,
         "mix": 10},
        # half of each of these caches is dropped
        {"name": "evict_half", "kind": "evict", "B": 16, "HKV": 8, "N": 4096, "D": 128, "lo": 1024, "budget": 2048,
         "recent": 256, "capacity": 2304, "mix": 11},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["train", "train", "train", "prefill", "prefill", "decode", "decode", "kv8_step", "kv8_step",
                       "kv8_prompts", "weighted", "evict"])
    hq, hkv = rng.choice([(8, 8), (16, 16), (32, 8), (32, 8), (32, 4), (64, 8), (12, 4)])
    mix = rng.randint(100, 99999)
    if kind in ("train", "prefill"):
        dtype = rng.choice(["float16", "float16", "float32"]) if kind == "train" else "float16"
        d = rng.choice([64, 64, 80, 96, 128, 128] if kind == "train" else [64, 80, 128, 128, 256])
        n = _log_int(rng, 32, 2048 if kind == "train" else 8192)
        pair = hq * d * n * n * 1.0
        budget = (2e10 if kind == "train" else 6e10) * (1.0 if dtype == "float16" else 0.2)
        if pair > budget:
            n = max(32, int(n * math.sqrt(budget / pair)))
            pair = hq * d * n * n * 1.0
        b = max(1, min(_log_int(rng, 1, 8), int(budget / pair)))
        causal = rng.random() < 0.75
        cap = rng.choice([0.0, 0.0, 20.0, 30.0, 50.0])
        bias = rng.random() < 0.4
        docs = _log_int(rng, 16, max(17, n)) if rng.random() < 0.5 else 0
        prefix = rng.randint(1, n) if causal and rng.random() < 0.3 else 0
        case = {"kind": kind, "B": b, "HQ": hq, "HKV": hkv, "N": n, "D": d, "causal": causal, "cap": cap,
                "bias": bias, "docs": docs, "prefix": prefix, "mix": mix}
        if kind == "train":
            case["dtype"] = dtype
        return case
    d = rng.choice([64, 80, 128, 128, 128, 256])
    n = _log_int(rng, 64, 32768)
    b = max(1, min(_log_int(rng, 1, 128), int(3e8 / (4.0 * hkv * n * d))))
    if kind in ("decode", "weighted"):
        case = {"kind": kind, "B": b, "HQ": hq, "HKV": hkv, "N": n, "D": d, "lo": rng.randint(0, n // 4), "mix": mix}
        if kind == "decode":
            case.update(cap=rng.choice([0.0, 30.0, 50.0]), bias=rng.random() < 0.5)
        return case
    codes, page = rng.choice(["int8", "e4m3"]), rng.choice([16, 16, 32, 64])
    if kind == "kv8_step":
        return {"kind": kind, "codes": codes, "B": b, "HQ": hq, "HKV": hkv, "hi": n, "D": d, "lo": rng.randint(1, n),
                "page": page, "cap": rng.choice([0.0, 0.0, 50.0]), "mix": mix}
    if kind == "kv8_prompts":
        hi = min(n, 4096)
        b = max(1, min(_log_int(rng, 1, 32), int(3e7 / (hkv * hi * d))))
        return {"kind": kind, "codes": codes, "B": b, "HKV": hkv, "lo": rng.randint(1, hi), "hi": hi, "D": d,
                "page": page, "mix": mix}
    budget = rng.randint(max(1, n // 8), n)
    return {"kind": kind, "B": b, "HKV": hkv, "N": n, "D": d, "lo": rng.randint(0, n), "budget": budget,
            "recent": rng.randint(0, budget), "capacity": budget + rng.randint(0, 256), "mix": mix}


# ---------------------------------------------------------------- what a case stands for


def _lengths(case):
    """A ragged batch's lengths, uniform in [lo, hi] with the longest one always there; ``mix``
    says which batch composition."""
    g = torch.Generator().manual_seed(case["mix"])
    hi = case["hi"] if "hi" in case else case["N"]
    lens = torch.randint(min(case["lo"], hi), hi + 1, (case["B"],), generator=g)
    lens[case["B"] // 2] = hi
    return lens


def _doc_ids(case):
    """Document of each position, [B, N]: lengths about ``docs``, a padded tail (id -1) in every other row."""
    if not case["docs"]:
        return None
    g = torch.Generator().manual_seed(case["mix"])
    n = case["N"]
    ids = torch.full((case["B"], n), -1, dtype=torch.int32)
    for b in range(case["B"]):
        end = n if b % 2 else n - n // 16
        at = i = 0
        while at < end:
            size = int(torch.randint(max(1, case["docs"] // 2), case["docs"] * 3 // 2 + 1, (1,), generator=g))
            ids[b, at:min(end, at + size)] = i
            at, i = at + size, i + 1
    return ids


def _prefix_lens(case):
    """Length of each row's prefix, up to ``prefix``."""
    if not case["prefix"]:
        return None
    g = torch.Generator().manual_seed(case["mix"])
    return torch.randint(0, case["prefix"] + 1, (case["B"],), generator=g, dtype=torch.int32)


def _pairs(case):
    """Visible (query, key) pairs of all rows of the batch."""
    n, ids, prefix, total = case["N"], _doc_ids(case), _prefix_lens(case), 0
    for b in range(case["B"]):
        pre = int(prefix[b]) if prefix is not None else 0
        segments = [(0, n)]
        if ids is not None:
            _, sizes = torch.unique_consecutive(ids[b], return_counts=True)
            ends = torch.cumsum(sizes, 0)
            segments = [(int(e - s), int(e)) for s, e in zip(sizes, ends) if int(ids[b, e - 1]) >= 0]
        for s, e in segments:
            m = e - s
            if not case["causal"]:
                total += m * m
                continue
            p = min(max(pre - s, 0), m)  # keys of the segment that every row of it sees
            total += m * (m + 1) // 2 + p * (p - 1) // 2
    return float(total)


def _slopes(heads):
    return torch.exp2(-8.0 * torch.arange(1, heads + 1, dtype=torch.float32) / heads)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape, dtype=HALF):
        return torch.randn(*shape, generator=g, device=dev, dtype=dtype)

    kind, b, d, hkv = case["kind"], case["B"], case["D"], case["HKV"]
    st = {"case": case, "slopes": None}
    if case.get("bias"):
        st["slopes"] = _slopes(case["HQ"]).to(dev)
    if kind in ("train", "prefill"):
        dtype = getattr(torch, case.get("dtype", "float16"))
        st["q"] = randn(b, case["HQ"], case["N"], d, dtype=dtype)
        st["k"] = randn(b, hkv, case["N"], d, dtype=dtype)
        st["v"] = randn(b, hkv, case["N"], d, dtype=dtype)
        ids, prefix = _doc_ids(case), _prefix_lens(case)
        st["ids"] = None if ids is None else ids.to(dev)
        st["prefix"] = None if prefix is None else prefix.to(dev)
        if kind == "train":
            st["dout"] = randn(b, case["HQ"], case["N"], d, dtype=dtype)
            for t in ("q", "k", "v"):
                st[t].requires_grad_()
    elif kind in ("decode", "weighted"):
        n = case["N"]
        st["q"] = randn(b, case["HQ"], 1, d)
        st["k"], st["v"] = randn(b, hkv, n, d), randn(b, hkv, n, d)
        # cache_lens is the current token's row, so a sequence of L tokens has L - 1
        st["cache_lens"] = (_lengths(case).clamp(min=1) - 1).to(torch.int32).to(dev)
        if kind == "weighted":
            st["weight"] = torch.rand(b, hkv, n, generator=g, device=dev)
            st["weight_out"] = torch.zeros_like(st["weight"])
    elif kind in ("kv8_step", "kv8_prompts"):
        page, top = case["page"], CODE_MAX[case["codes"]]
        lens = _lengths(case)
        blocks = (case["hi"] + page - 1) // page
        pages = b * blocks
        for t in ("k", "v"):
            # a page's largest of 16 D values is about 3.5 standard deviations
            scale = (3.5 + 0.3 * randn(pages, hkv, dtype=torch.float32)).clamp(min=2.5) / top
            x = randn(pages, hkv, page, d)
            x.mul_(top / 3.5)
            if case["codes"] == "int8":
                st[t + "_cache"] = x.round_().clamp_(-top, top).to(torch.int8)
            else:
                st[t + "_cache"] = x.clamp_(-top, top).to(E4M3)
            st[t + "_scale"] = scale
        perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))
        st["table"] = perm.to(torch.int32).view(b, blocks).to(dev)
        new = torch.ones(b, dtype=torch.int64) if kind == "kv8_step" else lens
        old = lens - 1 if kind == "kv8_step" else torch.zeros_like(lens)
        cu = torch.zeros(b + 1, dtype=torch.int32)
        cu[1:] = torch.cumsum(new, 0)
        st["cu"], st["max_new"] = cu.to(dev), int(new.max())
        st["old_lens"] = old.to(torch.int32).to(dev)
        st["seq_lens"] = lens.to(torch.int32).to(dev)
        st["k_new"], st["v_new"] = (randn(int(cu[-1]), hkv, d) for _ in range(2))
        if kind == "kv8_step":
            st["q"] = randn(b, case["HQ"], 1, d)
    else:  # evict: what tokens have been attended with is far from even
        n = case["N"]
        st["k"], st["v"] = randn(b, hkv, n, d), randn(b, hkv, n, d)
        st["weight"] = torch.empty(b, hkv, n, device=dev).exponential_(generator=g).pow_(3)
        st["seq_lens"] = _lengths(case).to(torch.int32).to(dev)
    return st


# ---------------------------------------------------------------- the operators in plain operations


def _plain_visible(st, b, n):
    case, dev = st["case"], st["q"].device
    i = torch.arange(n, device=dev)
    see = torch.ones(n, n, dtype=torch.bool, device=dev)
    if case["causal"]:
        see = i[None, :] <= i[:, None]
        if st["prefix"] is not None:
            see = see | (i[None, :] < st["prefix"][b])
    if st["ids"] is not None:
        ids = st["ids"][b]
        see = see & (ids[None, :] == ids[:, None]) & (ids >= 0)[None, :]
    return see


def _plain_scores(q, k, cap, slopes, dist):
    """Scores before the mask of heads q [G, M, D] on keys k [N, D], and the capped ones before the bias."""
    s = torch.matmul(q, k.t().contiguous()) * (1.0 / math.sqrt(q.shape[-1]))
    if cap:
        s = cap * torch.tanh(s / cap)
    return (s if slopes is None else s - slopes[:, None, None] * dist), s


def _plain_softmax(s, see):
    s = s.masked_fill(~see, -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    e = torch.exp(s - top)
    return e / torch.clamp(e.sum(-1, keepdim=True), min=1e-30)


def _plain_attention(st):
    case = st["case"]
    n, group, cap, train = case["N"], case["HQ"] // case["HKV"], case["cap"], case["kind"] == "train"
    q, k, v = (st[t].detach() for t in ("q", "k", "v"))
    i = torch.arange(n, device=q.device, dtype=torch.float32)
    dist = (i[None, :] - i[:, None]).abs() if case["bias"] else None
    out = torch.empty_like(q)
    dq, dk, dv = (torch.empty_like(t) for t in (q, k, v)) if train else (None, None, None)
    scale = 1.0 / math.sqrt(case["D"])
    for b in range(case["B"]):
        see = _plain_visible(st, b, n)
        for h in range(case["HKV"]):
            heads = slice(h * group, (h + 1) * group)
            slopes = None if st["slopes"] is None else st["slopes"][heads]
            kf, vf, qf = k[b, h].float(), v[b, h].float(), q[b, heads].float()
            s, capped = _plain_scores(qf, kf, cap, slopes, dist)
            p = _plain_softmax(s, see)
            del s
            o = torch.matmul(p, vf)
            out[b, heads] = o.to(out.dtype)
            if not train:
                continue
            do = st["dout"][b, heads].float()
            ds = torch.matmul(do, vf.t().contiguous())
            ds = p * (ds - (do * o).sum(-1, keepdim=True))
            if cap:
                ds = ds * (1.0 - (capped / cap) ** 2)
            dv[b, h] = torch.matmul(p.transpose(1, 2).contiguous(), do).sum(0).to(dv.dtype)
            dq[b, heads] = (torch.matmul(ds, kf) * scale).to(dq.dtype)
            dk[b, h] = (torch.matmul(ds.transpose(1, 2).contiguous(), qf).sum(0) * scale).to(dk.dtype)
    return {"out": out, "dq": dq, "dk": dk, "dv": dv} if train else out


def _plain_attend_one(q, k, v, cap, slopes):
    """One token: q [HQ, D] on k, v [HKV, L, D] in 32 bits -> (o [HQ, D], p [HQ, L])."""
    group = q.shape[0] // k.shape[0]
    n = k.shape[1]
    dist = (n - 1) - torch.arange(n, device=q.device, dtype=torch.float32)
    qg = q.view(k.shape[0], group, -1)
    s = torch.matmul(qg, k.transpose(1, 2).contiguous()) * (1.0 / math.sqrt(q.shape[-1]))
    if cap:
        s = cap * torch.tanh(s / cap)
    if slopes is not None:
        s = s - slopes.view(k.shape[0], group, 1) * dist
    e = torch.exp(s - s.amax(-1, keepdim=True))
    p = e / e.sum(-1, keepdim=True)
    return torch.matmul(p, v).reshape(q.shape[0], -1), p


def _plain_decode(st):
    case = st["case"]
    out = torch.empty_like(st["q"])
    weight = None
    if case["kind"] == "weighted":
        weight = st["weight_out"]
    for b, last in enumerate(st["cache_lens"].tolist()):
        n = min(last + 1, case["N"])
        o, p = _plain_attend_one(st["q"][b, :, 0].float(), st["k"][b, :, :n].float(), st["v"][b, :, :n].float(),
                                 case.get("cap", 0.0), st["slopes"])
        out[b, :, 0] = o.to(out.dtype)
        if weight is not None:
            weight[b, :, :n] = st["weight"][b, :, :n] + p.sum(1)
    return out if weight is None else {"out": out, "weight": weight}


def _plain_codes(x, scale, codes):
    """x [H, T, D] in 32 bits as codes of scale [H]."""
    top = CODE_MAX[codes]
    s = scale[:, None, None]
    y = torch.where(s > 0, x / s, torch.zeros_like(x)).clamp(-top, top)
    return y.round().to(torch.int8) if codes == "int8" else y.to(E4M3)


def _plain_append(st):
    case = st["case"]
    page, top = case["page"], CODE_MAX[case["codes"]]
    cu, old, table = st["cu"].tolist(), st["old_lens"].tolist(), st["table"].tolist()
    for b in range(case["B"]):
        at, end = old[b], old[b] + cu[b + 1] - cu[b]
        while at < end:
            upto = min(end, (at // page + 1) * page)
            pg, first = table[b][at // page], at % page
            rows = slice(cu[b] + at - old[b], cu[b] + upto - old[b])
            for t in ("k", "v"):
                x = st[t + "_new"][rows].float().transpose(0, 1)
                cache, scales = st[t + "_cache"], st[t + "_scale"]
                scale = x.abs().amax((1, 2)) / top
                if first:
                    before = scales[pg].clone()
                    scale = torch.maximum(scale, before)
                    kept = cache[pg, :, :first].float() * before[:, None, None]
                    again = _plain_codes(kept, scale, case["codes"])
                    grown = (scale > before)[:, None, None]
                    cache[pg, :, :first] = torch.where(grown, again.float(), cache[pg, :, :first].float()).to(cache.dtype)
                cache[pg, :, first:first + upto - at] = _plain_codes(x, scale, case["codes"])
                scales[pg] = scale
            at = upto
    return {t: st[t] for t in ("k_cache", "v_cache", "k_scale", "v_scale")}


def _plain_paged_decode(st):
    case = st["case"]
    page = case["page"]
    out = torch.empty_like(st["q"])
    for b, n in enumerate(st["seq_lens"].tolist()):
        ids = st["table"][b, :(n + page - 1) // page].long()
        kv = []
        for t in ("k", "v"):
            x = st[t + "_cache"][ids].float() * st[t + "_scale"][ids][:, :, None, None]
            kv.append(x.transpose(0, 1).reshape(case["HKV"], -1, case["D"])[:, :n])
        o, _ = _plain_attend_one(st["q"][b, :, 0].float(), kv[0], kv[1], case["cap"], st["slopes"])
        out[b, :, 0] = o.to(out.dtype)
    return out


def _plain_evict(st):
    case = st["case"]
    b, hkv, d, cap = case["B"], case["HKV"], case["D"], case["capacity"]
    dev = st["k"].device
    k_out, v_out = (torch.zeros(b, hkv, cap, d, dtype=HALF, device=dev) for _ in range(2))
    weight = torch.zeros(b, hkv, cap, device=dev)
    index = torch.full((b, hkv, cap), -1, dtype=torch.int32, device=dev)
    for i, n in enumerate(st["seq_lens"].tolist()):
        m = min(n, case["budget"])
        keep = torch.arange(n, device=dev).expand(hkv, n)
        if n > m:
            head = n - case["recent"]
            order = torch.sort(st["weight"][i, :, :head], dim=1, descending=True, stable=True)[1]
            heavy = torch.sort(order[:, :m - case["recent"]], dim=1)[0]
            keep = torch.cat([heavy, torch.arange(head, n, device=dev).expand(hkv, -1)], 1)
        index[i, :, :m] = keep.to(torch.int32)
        weight[i, :, :m] = torch.gather(st["weight"][i], 1, keep)
        rows = keep[:, :, None].expand(hkv, m, d)
        k_out[i, :, :m] = torch.gather(st["k"][i], 1, rows)
        v_out[i, :, :m] = torch.gather(st["v"][i], 1, rows)
    return [k_out, v_out, weight, index, st["seq_lens"].clamp(max=case["budget"])]


# ---------------------------------------------------------------- one pass


def run(st):
    case = st["case"]
    kind = case["kind"]
    if not own:
        if kind in ("train", "prefill"):
            return _plain_attention(st)
        if kind in ("decode", "weighted"):
            return _plain_decode(st)
        if kind == "kv8_prompts":
            return _plain_append(st)
        if kind == "kv8_step":
            caches = _plain_append(st)
            return {"out": _plain_paged_decode(st), **caches}
        return _plain_evict(st)
    import flash_attn_v100 as fa

    if kind == "train":
        from flash_attn_autograd import flash_attn_scored

        out = flash_attn_scored(st["q"], st["k"], st["v"], case["causal"], case["cap"], st["slopes"], st["ids"],
                                st["prefix"])
        dq, dk, dv = torch.autograd.grad(out, (st["q"], st["k"], st["v"]), st["dout"])
        return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}
    if kind == "prefill":
        return fa.forward_scored(st["q"], st["k"], st["v"], case["causal"], case["cap"], st["slopes"], st["ids"],
                                 st["prefix"])
    if kind == "decode":
        return fa.forward_decode_scored_gqa_fp16(st["q"], st["k"], st["v"], st["cache_lens"], case["cap"],
                                                 st["slopes"])
    if kind == "weighted":
        out, weight = fa.forward_decode_weighted_gqa_fp16(st["q"], st["k"], st["v"], st["cache_lens"], st["weight"],
                                                          st["weight_out"])
        return {"out": out, "weight": weight}
    if kind in ("kv8_step", "kv8_prompts"):
        fa.append_paged_kv8(st["k_new"], st["v_new"], st["cu"], st["old_lens"], st["max_new"], st["k_cache"],
                            st["v_cache"], st["k_scale"], st["v_scale"], st["table"])
        caches = {t: st[t] for t in ("k_cache", "v_cache", "k_scale", "v_scale")}
        if kind == "kv8_prompts":
            return caches
        out = fa.forward_paged_decode_kv8_gqa(st["q"], st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"],
                                              st["table"], st["seq_lens"], case["cap"], st["slopes"])
        return {"out": out, **caches}
    return list(fa.evict_by_weight(st["k"], st["v"], st["weight"], st["seq_lens"], case["budget"], case["recent"],
                                   case["capacity"]))


def work(case):
    kind, b, d, hkv = case["kind"], case["B"], case["D"], case["HKV"]
    if kind in ("train", "prefill"):
        size = 4 if case.get("dtype") == "float32" else 2
        hq, n, pairs = case["HQ"], case["N"], _pairs(case)
        rows = (2.0 * hq + 2.0 * hkv) * b * n * d * size  # q, k, v in, out
        if kind == "prefill":
            return {"bytes": rows, "flops": 4.0 * hq * d * pairs}
        # forward, then dout, q, k, v, out in, dq, dk, dv out: two products forward, five backward
        return {"bytes": rows + (4.0 * hq + 4.0 * hkv) * b * n * d * size, "flops": 14.0 * hq * d * pairs}
    tokens = float(_lengths(case).sum())
    if kind in ("decode", "weighted"):
        tokens = float(_lengths(case).clamp(min=1).sum())
        extra = 8.0 * hkv * tokens if kind == "weighted" else 0.0
        return {"bytes": tokens * hkv * 4.0 * d + 4.0 * b * case["HQ"] * d + extra,
                "flops": 4.0 * case["HQ"] * d * tokens}
    if kind == "kv8_step":
        pages = tokens / case["page"]
        return {"bytes": 2.0 * hkv * (tokens * d + pages * 4.0) + b * (4.0 * case["HQ"] * d + 6.0 * hkv * d),
                "flops": 4.0 * case["HQ"] * d * tokens}
    if kind == "kv8_prompts":
        return {"bytes": 2.0 * hkv * tokens * d * 3.0, "flops": 4.0 * hkv * tokens * d}
    kept = float(_lengths(case).clamp(max=case["budget"]).sum())
    written = float(b * case["capacity"])
    return {"bytes": hkv * (4.0 * tokens + kept * 4.0 * d + written * (4.0 * d + 8.0)), "flops": hkv * tokens}


# ---------------------------------------------------------------- the definitions in 64 bits


def _exact_head(q, k, v, see, cap, slope, dist):
    """Outputs of query heads q [G, M, D] over one KV head, differentiable."""
    s = q @ k.t() / math.sqrt(q.shape[-1])
    if cap:
        s = cap * torch.tanh(s / cap)
    if slope is not None:
        s = s - slope.view(-1, 1, 1) * dist
    s = torch.where(see, s, torch.full((), -1e300, dtype=s.dtype, device=s.device))
    top = s.detach().amax(-1, keepdim=True)
    w = torch.exp(s - top) * see
    total = w.sum(-1, keepdim=True)
    p = w / torch.where(total > 0, total, torch.ones_like(total))
    return p @ v, p


def _exact_attention(case, st):
    n, group = case["N"], case["HQ"] // case["HKV"]
    dev = st["q"].device
    pos = torch.arange(n, device=dev)
    dist = (pos[:, None] - pos[None, :]).abs().double()
    outs = {t: [] for t in ("out", "dq", "dk", "dv")}
    for b in range(case["B"]):
        see = torch.ones(n, n, dtype=torch.bool, device=dev)
        if case["causal"]:
            last = pos if st["prefix"] is None else torch.maximum(pos, st["prefix"][b] - 1)
            see &= pos[None, :] <= last[:, None]
        if st["ids"] is not None:
            ids = st["ids"][b]
            see &= (ids[:, None] == ids[None, :]) & (ids[:, None] >= 0)
        for h in range(case["HKV"]):
            heads = slice(h * group, (h + 1) * group)
            slope = None if st["slopes"] is None else st["slopes"][heads].double()
            k, v = st["k"][b, h].detach().double(), st["v"][b, h].detach().double()
            q = st["q"][b, heads].detach().double()
            if case["kind"] == "prefill":
                outs["out"].extend(_exact_head(q[i:i + 1], k, v, see, case["cap"],
                                               None if slope is None else slope[i:i + 1], dist)[0][0]
                                   for i in range(group))
                continue
            q, k, v = (t.requires_grad_() for t in (q, k, v))
            o, _ = _exact_head(q, k, v, see, case["cap"], slope, dist)
            dq, dk, dv = torch.autograd.grad(o, (q, k, v), st["dout"][b, heads].double())
            outs["out"].extend(o.detach())
            outs["dq"].extend(dq)
            outs["dk"].append(dk)
            outs["dv"].append(dv)
    if case["kind"] == "prefill":
        return torch.stack(outs["out"]).view(st["q"].shape)
    return {t: torch.stack(x).view(st["q" if t in ("out", "dq") else "k"].shape) for t, x in outs.items()}


def _exact_one(q, k, v, cap, slopes):
    """One token's heads q [HQ, D] over k, v [HKV, L, D]."""
    group, n = q.shape[0] // k.shape[0], k.shape[1]
    dist = torch.arange(n - 1, -1, -1, device=q.device).double()
    see = torch.ones(1, n, dtype=torch.bool, device=q.device)
    got = []
    for h in range(k.shape[0]):
        heads = slice(h * group, (h + 1) * group)
        slope = None if slopes is None else slopes[heads].double()
        got.append(_exact_head(q[heads, None].double(), k[h].double(), v[h].double(), see, cap, slope, dist))
    return torch.cat([o[:, 0] for o, _ in got]), torch.stack([p[:, 0].sum(0) for _, p in got])


def _exact_evict(case, st):
    """The rows by (weight, lower index first) of each head, on the host."""
    shape = (case["B"], case["HKV"], case["capacity"])
    index = np.full(shape, -1, dtype=np.int32)
    lens = st["seq_lens"].cpu().numpy()
    weight = st["weight"].double().cpu().numpy()
    for b, h in np.ndindex(*shape[:2]):
        head = max(0, int(lens[b]) - case["recent"]) if lens[b] > case["budget"] else 0
        order = np.lexsort((np.arange(head), -weight[b, h, :head]))
        heavy = np.sort(order[:case["budget"] - case["recent"]])
        rows = np.concatenate([heavy, np.arange(head, lens[b])])
        index[b, h, :rows.size] = rows
    index = torch.from_numpy(index).to(st["k"].device)
    live, rows = index >= 0, index.clamp(min=0).long()

    def take(x):
        at = rows if x.dim() == 3 else rows[..., None].expand(*rows.shape, x.shape[-1])
        got = torch.gather(x, 2, at).double()
        return got * (live if x.dim() == 3 else live[..., None])

    return [take(st["k"]), take(st["v"]), take(st["weight"]), index, st["seq_lens"].clamp(max=case["budget"])]


def exact(case, seed):
    kind = case["kind"]
    if kind in ("train", "prefill"):
        return _exact_attention(case, prepare(case, seed))
    st = prepare(case, seed)
    if kind == "evict":
        return _exact_evict(case, st)
    if kind in ("decode", "weighted"):
        out = torch.empty(st["q"].shape, dtype=torch.float64, device=st["q"].device)
        weight = torch.zeros(st["k"].shape[:3], dtype=torch.float64, device=out.device)
        for b, last in enumerate(st["cache_lens"].tolist()):
            n = min(last + 1, case["N"])
            out[b, :, 0], p = _exact_one(st["q"][b, :, 0], st["k"][b, :, :n], st["v"][b, :, :n], case.get("cap", 0.0),
                                         st["slopes"])
            if kind == "weighted":
                weight[b, :, :n] = st["weight"][b, :, :n].double() + p
        return {"out": out, "weight": weight} if kind == "weighted" else out
    # codes are whole numbers of a quotient rounded in 32 bits and have no value in 64; scales do
    top, page = CODE_MAX[case["codes"]], case["page"]
    scales = {t: st[t + "_scale"].double() for t in ("k", "v")}
    cu, old = st["cu"].tolist(), st["old_lens"].tolist()
    for b in range(case["B"]):
        for first in range(old[b] // page * page, old[b] + cu[b + 1] - cu[b], page):
            a, z = max(first, old[b]) - old[b] + cu[b], min(first + page, old[b] + cu[b + 1] - cu[b]) - old[b] + cu[b]
            pg = int(st["table"][b, first // page])
            for t in ("k", "v"):
                s = st[t + "_new"][a:z].double().abs().amax((0, 2)) / top
                scales[t][pg] = torch.maximum(s, scales[t][pg]) if first < old[b] else s
    state = {"k_cache": None, "v_cache": None, "k_scale": scales["k"], "v_scale": scales["v"]}
    if kind == "kv8_prompts":
        return state
    _plain_append(st)  # the codes by their definition
    out = torch.empty(st["q"].shape, dtype=torch.float64, device=st["q"].device)
    for b, n in enumerate(st["seq_lens"].tolist()):
        pg = st["table"][b, torch.arange(n, device=out.device) // page].long()
        row = torch.arange(n, device=out.device) % page
        kv = [(st[t + "_cache"].view(torch.uint8)[pg, :, row].view(st[t + "_cache"].dtype).float().double() *
               st[t + "_scale"].double()[pg][:, :, None]).transpose(0, 1) for t in ("k", "v")]
        out[b, :, 0], _ = _exact_one(st["q"][b, :, 0], kv[0], kv[1], case["cap"], st["slopes"])
    return {"out": out, **state}
