"""Single-token attention with modified scores, the 8-bit paged cache with page
scales, the decode that adds up attention weights and the eviction by them:
against the oracle (64 bits; codes, indexes and copies exactly), at the lengths,
pages and layouts where they can go wrong, and the calls that are refused.

Bounds, u = 2^-24, h = 2^-11 (half a step of fp16), n keys:
  score |dy| <= (D + 16) u sum_d |q_d k_d| / sqrt(D) + 8 u (|y| + slope distance)
  P     |dP| <= P (|dy| + max |dy| + 2 (n + 16) u)
  O     |dO| <= (dP + (h + (n + 16) u) P) |V| + n 2^-25 max |V| + h |O|
        (h P: probabilities, times the V scale, rounded to fp16 against a running
        reference; the n 2^-25 term: those that fall below fp16's normal numbers)
  weights: |dP| of the heads, and 2 (G + 1) u of the sum
"""
import math

import pytest
import torch

from oracle import attention as A
from tests.helpers import randn

pytestmark = pytest.mark.gpu
F16, F32, I8, F8 = torch.float16, torch.float32, torch.int8, torch.float8_e4m3fn
U, H = 2.0 ** -24, 2.0 ** -11


def gen(seed):
    return torch.Generator().manual_seed(seed)


def slopes_of(h):
    return torch.exp2(-8.0 * torch.arange(1, h + 1, dtype=F32) / h)


def bounds(q, k, v, lens, cap, slopes):
    """Oracle and error bounds of the output and the probabilities for rows k, v [B, H_KV, N, D]."""
    ro, p, y = A.scored_decode(q, k, v, lens, cap, slopes)
    b, hq, _, d = q.shape
    n = k.shape[2]
    live = torch.arange(n)[None, :] < torch.as_tensor([int(x) for x in lens])[:, None]
    clean = lambda t: torch.where(live[:, None, :, None], t.double(), torch.zeros((), dtype=torch.float64))
    ke, ve = A.expand_kv(clean(k), hq), A.expand_kv(clean(v), hq)
    dist = 0.0
    if slopes is not None:
        dist = slopes.double().abs()[None, :, None] * torch.arange(n).double()[None, None, :].flip(-1)
    dy = (d + 16) * U * (ke.abs() @ q[:, :, 0].double().abs()[..., None])[..., 0] / math.sqrt(d) + 8 * U * (y.abs() + dist)
    dy = dy * live[:, None]
    dp = p * (dy + dy.amax(-1, keepdim=True) + 2 * (n + 16) * U)
    bo = ((dp + (H + (n + 16) * U) * p)[:, :, None] @ ve.abs())
    bo = (bo + n * 2.0 ** -25 * ve.abs().amax((-2, -1), keepdim=True)) * (1 + H) + H * ro.abs() + 2.0 ** -25
    return ro, bo, p, dp


def check(what, got, ref, bound):
    got = got.detach().double().cpu()
    assert got.shape == ref.shape and bool(torch.isfinite(got).all()), what
    over = (got - ref).abs() - bound
    worst = int(over.argmax())
    assert over.max() <= 0, (f"{what}: {int((over > 0).sum())} of {over.numel()} past the bound; worst {got.flatten()[worst]:.6g} "
                             f"for {ref.flatten()[worst]:.6g}, bound {bound.flatten()[worst]:.3g}")


def ragged(g, b, n, lo=0):
    """Numbers of rows, 0 and n among them where they fit."""
    lens = torch.randint(lo, n + 1, (b,), generator=g)
    lens[0] = n
    if b > 2 and lo == 0:
        lens[1], lens[2] = 0, 1
    return lens


#        b hq hkv n     d
DECODE = [(1, 1, 1, 1, 64), (3, 4, 2, 17, 128), (2, 8, 8, 33, 64), (5, 32, 8, 300, 128), (2, 6, 1, 129, 80),
          (3, 16, 1, 250, 256), (2, 48, 2, 200, 64), (2, 4, 4, 100, 100), (3, 5, 1, 77, 33), (1, 32, 8, 4097, 128),
          (40, 16, 4, 700, 96), (2, 8, 2, 3000, 192), (70, 8, 2, 2500, 64), (130, 8, 8, 300, 128), (300, 8, 2, 260, 64)]


@pytest.mark.parametrize("cap,bias", [(0.0, False), (5.0, False), (0.0, True), (30.0, True)])
@pytest.mark.parametrize("b,hq,hkv,n,d", DECODE)
def test_scored_decode(fa, b, hq, hkv, n, d, cap, bias):
    """Rows past a sequence's end hold NaN."""
    g = gen(b + n + d)
    q, k, v = randn(g, b, hq, 1, d) * 2, randn(g, b, hkv, n, d), randn(g, b, hkv, n, d)
    lens = ragged(g, b, n)
    slopes = slopes_of(hq) if bias else None
    ro, bo, _, _ = bounds(q, k, v, lens, cap, slopes)
    dead = torch.arange(n)[None, :] >= lens[:, None]
    for t in (k, v):
        t.masked_fill_(dead[:, None, :, None], math.nan)
    dev = None if slopes is None else slopes.cuda()
    out = fa.forward_decode_scored_gqa_fp16(q.cuda(), k.cuda(), v.cuda(), (lens - 1).int().cuda(), cap, dev)
    check("out", out, ro, bo)
    # lengths past the cache attend all of it
    k, v = (torch.nan_to_num(t) for t in (k, v))
    over = torch.full((b,), n + 5, dtype=torch.int32, device="cuda")
    full = fa.forward_decode_scored_gqa_fp16(q.cuda(), k.cuda(), v.cuda(), over, cap, dev)
    same = fa.forward_decode_scored_gqa_fp16(q.cuda(), k.cuda(), v.cuda(), torch.full_like(over, n - 1), cap, dev)
    assert torch.equal(full, same)


def test_scored_decode_agrees_with_plain_decode(fa):
    g = gen(8)
    q, k, v = randn(g, 6, 32, 1, 128), randn(g, 6, 8, 900, 128), randn(g, 6, 8, 900, 128)
    lens = (ragged(g, 6, 900, 1) - 1).int().cuda()
    a = fa.forward_decode_scored_gqa_fp16(q.cuda(), k.cuda(), v.cuda(), lens)
    r = fa.forward_continuous_batching_fp16(q.cuda(), k.cuda(), v.cuda(), lens, True)
    assert (a.float() - r.float()).abs().max() <= 2e-3


def test_unaligned_cache(fa):
    g = gen(12)
    q, k, v = randn(g, 2, 4, 1, 64), randn(g, 2, 2, 200, 64), randn(g, 2, 2, 200, 64)
    shift = lambda t: torch.cat([torch.zeros(1, dtype=t.dtype), t.flatten()]).cuda()[1:].view(t.shape)
    lens = torch.tensor([199, 120], dtype=torch.int32)
    ro, bo, _, _ = bounds(q, k, v, lens + 1, 9.0, None)
    check("out", fa.forward_decode_scored_gqa_fp16(shift(q), shift(k), shift(v), lens.cuda(), 9.0), ro, bo)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("b,hq,hkv,n,d", DECODE)
def test_weighted_decode(fa, b, hq, hkv, n, d, in_place):
    g = gen(b * 3 + n + d)
    q, k, v = randn(g, b, hq, 1, d) * 2, randn(g, b, hkv, n, d), randn(g, b, hkv, n, d)
    lens = ragged(g, b, n)
    weight = torch.rand(b, hkv, n, generator=g)
    for cap, slopes in ((0.0, None), (6.0, slopes_of(hq))):
        ro, bo, p, dp = bounds(q, k, v, lens, cap, slopes)
        w = weight.cuda()
        target = w if in_place else torch.full_like(w, -3.0)
        sl = None if slopes is None else slopes.cuda()
        out, got = fa.forward_decode_weighted_gqa_fp16(q.cuda(), k.cuda(), v.cuda(), (lens - 1).int().cuda(), w,
                                                       None if in_place else target, cap, sl)
        assert got.data_ptr() == target.data_ptr()
        check("out", out, ro, bo)
        group = lambda t: t.view(b, hkv, hq // hkv, n).sum(2)
        ref = weight.double() + group(p)
        live = (torch.arange(n)[None, :] < lens[:, None])[:, None]
        untouched = weight.double() if in_place else torch.full_like(ref, -3.0)
        # the log-sum-exp of each split is rounded once more, and log2 to 4 u of its value
        bound = group(dp + p * 64 * U) + 2 * (hq // hkv + 1) * U * ref
        check("weight", got, torch.where(live, ref, untouched), torch.where(live, bound, torch.zeros_like(bound)))
        plain = fa.forward_decode_scored_gqa_fp16(q.cuda(), k.cuda(), v.cuda(), (lens - 1).int().cuda(), cap, sl)
        assert torch.equal(out, plain)


# ---------------------------------------------------------------- the 8-bit paged cache


def make_cache(g, dtype, pages, h, page, d):
    """Codes and scales with garbage everywhere: what a fresh allocation may hold."""
    raw = torch.randint(0, 256, (pages, h, page, d), generator=g).to(torch.uint8)
    scale = torch.rand(pages, h, generator=g)
    return raw.view(dtype), scale


def same_codes(a, b):
    """Equal codes; a NaN is any NaN (the sign that one takes through arithmetic is not specified, IEEE 754 6.3)."""
    raw = [t.cpu().contiguous().view(torch.uint8) for t in (a, b)]
    if a.dtype == F8:
        raw = [torch.where(x & 0x7f == 0x7f, torch.full_like(x, 0x7f), x) for x in raw]
    return torch.equal(*raw)


def run_append(fa, new_k, new_v, cu, lens, max_new, caches, table):
    """Appends on the GPU and by the oracle; both must hold the same codes and scales."""
    dev = [t.cuda() for t in caches]
    fa.append_paged_kv8(new_k.cuda(), new_v.cuda(), cu.cuda(), lens.cuda(), max_new, *dev, table.cuda())
    ref = A.append_paged_kv8(new_k, new_v, cu, lens, max_new, *caches, table)
    for name, a, r in zip(("k_cache", "v_cache"), dev, ref):
        assert same_codes(a, r), (name, int((a.cpu().view(torch.uint8) != r.view(torch.uint8)).sum()))
    for a, r in zip(dev[2:], ref[2:]):
        assert torch.equal(a.cpu(), r)
    return dev, ref


@pytest.mark.parametrize("dtype", [I8, F8])
@pytest.mark.parametrize("h,page,d", [(2, 16, 128), (1, 16, 64), (3, 32, 80), (2, 64, 256), (2, 16, 36), (1, 128, 64),
                                      (1, 256, 256), (2, 16, 1)])
def test_append(fa, dtype, h, page, d):
    """Prompts, then single and several tokens into partly filled pages; amplitudes that make scales grow and stay."""
    g = gen(page + d)
    lens = torch.tensor([0, 1, page - 1, page, page + 3, 3 * page - 1], dtype=torch.int32)
    b, blocks = len(lens), 6
    table = torch.randperm(b * blocks, generator=g).int().view(b, blocks)
    caches = make_cache(g, dtype, b * blocks, h, page, d)
    caches = (caches[0], make_cache(g, dtype, b * blocks, h, page, d)[0], caches[1], caches[1].flip(0).contiguous())
    empty = torch.zeros(b, dtype=torch.int32)
    for old, counts, amp in ((empty, lens.tolist(), 1.0), (lens, [1] * b, 0.3), (lens + 1, [2, 0, page, 1, 2 * page, 7], 4.0),
                             (lens + torch.tensor([3, 1, page + 1, 2, 2 * page + 1, 8]).int(), [1] * b, 0.0)):
        cu = torch.zeros(b + 1, dtype=torch.int32)
        cu[1:] = torch.cumsum(torch.tensor(counts), 0)
        nk, nv = (randn(g, int(cu[-1]), h, d) * amp for _ in range(2))
        if nk.shape[0] > 1:
            nv[1] *= 50.0
        dev, caches = run_append(fa, nk, nv, cu, old, max(counts) or 1, caches, table)


@pytest.mark.parametrize("dtype", [I8, F8])
def test_append_edges(fa, dtype):
    """Dropped tokens (bad pages, past the table, past max_new, negative lengths), zeros, the type's largest and least
    values; everything else stays as it was."""
    g = gen(4)
    h, page, d, blocks = 2, 16, 64, 3
    table = torch.tensor([[0, 1, 2], [3, -1, 99], [4, 5, 6], [7, 8, 9], [10, 11, 12], [13, 14, 15]], dtype=torch.int32)
    lens = torch.tensor([40, 10, -1, 5, 0, 47], dtype=torch.int32)
    counts = [20, 30, 4, 21, 9, 1]
    cu = torch.zeros(7, dtype=torch.int32)
    cu[1:] = torch.cumsum(torch.tensor(counts), 0)
    caches = make_cache(g, dtype, 16, h, page, d)
    caches = (caches[0], caches[0].flip(0).contiguous(), caches[1], caches[1] * 2)
    nk, nv = (randn(g, int(cu[-1]), h, d) for _ in range(2))
    nk[int(cu[4]):int(cu[5])] = 0.0
    nv[int(cu[4]):int(cu[5])] = 6e-8
    nk[int(cu[3]), 0, :3] = torch.tensor([65504.0, -65504.0, 1e-7], dtype=F16)
    run_append(fa, nk, nv, cu, lens, 20, caches, table)
    # boundaries that run past the packed rows, or backwards
    bad = torch.tensor([-5, 10, 8, 300, 200, 50, 60], dtype=torch.int32)
    run_append(fa, nk, nv, bad, lens.clamp(min=0), 20, caches, table)
    run_append(fa, nk[:0], nv[:0], torch.zeros(7, dtype=torch.int32), lens, 1, caches, table)


KV8 = [(1, 1, 1, 1, 16, 64), (3, 8, 2, 40, 16, 128), (2, 32, 8, 300, 16, 128), (2, 16, 1, 500, 32, 64), (3, 6, 2, 130, 64, 80),
       (2, 24, 1, 200, 16, 256), (1, 32, 8, 4100, 16, 128), (2, 4, 4, 90, 16, 40), (2, 3, 1, 70, 32, 33), (64, 32, 8, 700, 16, 128),
       (3, 8, 8, 1000, 256, 128), (70, 8, 2, 2500, 128, 64), (2, 8, 2, 9000, 16, 64), (3, 8, 4, 2000, 16, 192)]


@pytest.mark.parametrize("dtype", [I8, F8])
@pytest.mark.parametrize("b,hq,hkv,n,page,d", KV8)
def test_paged_kv8_decode(fa, dtype, b, hq, hkv, n, page, d):
    """Scattered pages; rows past the end, unused pages and their scales hold garbage and NaN; scales over six decades."""
    g = gen(b + n + d + page)
    lens = ragged(g, b, n)
    blocks = (n + page - 1) // page
    pages = b * blocks + 3
    table = torch.randperm(pages, generator=g)[:b * blocks].int().view(b, blocks)
    q = randn(g, b, hq, 1, d)
    codes = [make_cache(g, I8, pages, hkv, page, d)[0] for _ in range(2)]
    if dtype == F8:
        codes = [(c.float() * 3.5).to(F8) for c in codes]
    top = A.KV8_TOP[dtype]
    ks = (1 + torch.rand(pages, hkv, generator=g)) / top
    vs = torch.exp(torch.empty(pages, hkv).uniform_(math.log(1e-3), math.log(1e3), generator=g)) / top
    garbage = 0x80 if dtype == I8 else 0x7f  # -128, NaN
    used = torch.zeros(pages, dtype=torch.bool)
    for i in range(b):
        m = int(lens[i])
        used[table[i, :(m + page - 1) // page].long()] = True
        if m % page:  # the last page's rows past the end
            for c in codes:
                c.view(torch.uint8)[int(table[i, m // page]), :, m % page:] = garbage
    ks[~used], vs[~used] = math.nan, math.inf
    for c in codes:
        c.view(torch.uint8)[~used] = garbage
    k, v = A.paged_kv8_rows(codes[0], ks, table, lens), A.paged_kv8_rows(codes[1], vs, table, lens)
    table[~(torch.arange(blocks)[None, :] < (lens[:, None] + page - 1) // page)] = -7  # entries past the end are not read
    args = [t.cuda() for t in (q, *codes, ks, vs, table, lens.int())]
    for cap, slopes in ((0.0, None), (10.0, slopes_of(hq))):
        ro, bo, _, _ = bounds(q, k, v, lens, cap, slopes)
        out = fa.forward_paged_decode_kv8_gqa(*args, cap, None if slopes is None else slopes.cuda())
        check("out", out, ro, bo)


def test_paged_kv8_bad_pages(fa):
    g = gen(2)
    q = randn(g, 4, 4, 1, 64).cuda()
    codes, scale = make_cache(g, I8, 6, 2, 16, 64)
    codes, scale = codes.cuda(), scale.cuda()
    table = torch.tensor([[0, 1, 2], [0, 9, 2], [-1, 1, 2], [3, 4, 5]], dtype=torch.int32).cuda()
    lens = torch.tensor([48, 40, 1, 49], dtype=torch.int32).cuda()
    out = fa.forward_paged_decode_kv8_gqa(q, codes, codes, scale, scale, table, lens)
    bad = torch.isnan(out).all(-1).all(1)[:, 0].tolist()
    assert bad == [False, True, True, True] and bool(torch.isfinite(out[0]).all())
    out = fa.forward_paged_decode_kv8_gqa(q, codes, codes, scale, scale, table, lens.clamp(max=16) * 0)
    assert not out.any()
    none = fa.forward_paged_decode_kv8_gqa(q, codes[:0], codes[:0], scale[:0], scale[:0], table, lens)
    assert bool(torch.isnan(none).all())
    no_table = fa.forward_paged_decode_kv8_gqa(q, codes, codes, scale, scale, table[:, :0].contiguous(), lens)
    assert bool(torch.isnan(no_table).all())


@pytest.mark.parametrize("zero", ["some", "all"])
def test_pages_of_zeros(fa, zero):
    """A page whose tokens are all zero has scale 0."""
    g = gen(6)
    b, hq, hkv, page, d, n = 2, 4, 2, 16, 64, 60
    table = torch.arange(8, dtype=torch.int32).view(2, 4)
    nk, nv = randn(g, 2 * n, hkv, d), randn(g, 2 * n, hkv, d)
    (nv if zero == "all" else nv[:16]).zero_()
    nk[n:n + 16] = 0
    caches = [torch.zeros(8, hkv, page, d, dtype=I8) for _ in range(2)] + [torch.full((8, hkv), math.nan) for _ in range(2)]
    cu, lens = torch.tensor([0, n, 2 * n], dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    dev, ref = run_append(fa, nk, nv, cu, lens, n, caches, table)
    q = randn(g, b, hq, 1, d)
    full = torch.tensor([n, n], dtype=torch.int32)
    k, v = A.paged_kv8_rows(ref[0], ref[2], table, full), A.paged_kv8_rows(ref[1], ref[3], table, full)
    ro, bo, _, _ = bounds(q, k, v, full, 0.0, None)
    check("out", fa.forward_paged_decode_kv8_gqa(q.cuda(), *dev, table.cuda(), full.cuda()), ro, bo)


# ---------------------------------------------------------------- eviction


@pytest.mark.parametrize("b,h,n,d,budget,recent,capacity", [
    (1, 1, 1, 64, 1, 0, 1), (2, 2, 40, 64, 16, 4, 20), (3, 2, 300, 128, 100, 100, 100), (2, 1, 1025, 80, 512, 0, 600),
    (2, 3, 5000, 64, 1700, 33, 1800), (2, 2, 200, 33, 64, 10, 64), (3, 2, 100, 64, 300, 50, 310), (2, 2, 64, 64, 0, 0, 5),
    (1, 2, 33000, 8, 20000, 100, 20000)])
@pytest.mark.parametrize("pattern", ["heavy", "ties", "extremes"])
def test_evict(fa, b, h, n, d, budget, recent, capacity, pattern):
    g = gen(n + budget)
    k, v = randn(g, b, h, n, d), randn(g, b, h, n, d)
    if pattern == "heavy":
        weight = torch.empty(b, h, n).exponential_(generator=g) ** 3
    elif pattern == "ties":
        weight = torch.randint(0, 4, (b, h, n), generator=g).float() * 0.25
    else:
        vals = torch.tensor([-math.inf, -3.4e38, -1e-45, -0.0, 0.0, 1e-45, 1.0, 3.4e38, math.inf, math.nan])
        weight = vals[torch.randint(0, 10, (b, h, n), generator=g)]
    lens = ragged(g, b, n)
    lens[-1] = n
    got = fa.evict_by_weight(k.cuda(), v.cuda(), weight.cuda(), lens.int().cuda(), budget, recent, capacity)
    ref = A.evict_by_weight(k, v, weight, lens, budget, recent, capacity)
    for a, r in zip(got, ref):
        assert a.dtype == r.dtype and torch.equal(a.cpu().nan_to_num(nan=7.0) if a.is_floating_point() else a.cpu(),
                                                  r.nan_to_num(nan=7.0) if r.is_floating_point() else r)


def test_evict_reads_only_the_tokens_held(fa):
    g = gen(3)
    k, v = randn(g, 2, 2, 50, 64), randn(g, 2, 2, 50, 64)
    weight = torch.rand(2, 2, 50, generator=g)
    lens = torch.tensor([30, -4], dtype=torch.int32)
    ref = A.evict_by_weight(k, v, weight, lens, 20, 5, 25)
    weight[:, :, 30:] = math.inf
    k[:, :, 30:] = math.nan
    for a, r in zip(fa.evict_by_weight(k.cuda(), v.cuda(), weight.cuda(), lens.cuda(), 20, 5, 25), ref):
        assert torch.equal(a.cpu(), r)


# ---------------------------------------------------------------- as they are used


@pytest.mark.parametrize("dtype", [I8, F8])
def test_serving_on_the_8_bit_cache(fa, dtype):
    """A prompt and a few decoded tokens per sequence, through append and decode, one of the sequences idle."""
    g = gen(50)
    b, hq, hkv, page, d, blocks = 3, 8, 2, 16, 128, 8
    table = torch.randperm(b * blocks, generator=g).int().view(b, blocks)
    dev = [torch.zeros(b * blocks, hkv, page, d, dtype=dtype).cuda() for _ in range(2)] + [
        torch.zeros(b * blocks, hkv).cuda() for _ in range(2)]
    ref = [t.cpu() for t in dev]
    lens = torch.zeros(b, dtype=torch.int32)
    prompts = [37, 0, 64]
    for step in range(20):
        counts = prompts if step == 0 else [1, 0, 1]
        cu = torch.zeros(b + 1, dtype=torch.int32)
        cu[1:] = torch.cumsum(torch.tensor(counts), 0)
        nk, nv = (randn(g, int(cu[-1]), hkv, d) * (1 + 0.1 * step) for _ in range(2))
        fa.append_paged_kv8(nk.cuda(), nv.cuda(), cu.cuda(), lens.cuda(), max(counts), *dev, table.cuda())
        ref = A.append_paged_kv8(nk, nv, cu, lens, max(counts), *ref, table)
        lens = lens + torch.tensor(counts, dtype=torch.int32)
        q = randn(g, b, hq, 1, d)
        out = fa.forward_paged_decode_kv8_gqa(q.cuda(), *dev, table.cuda(), lens.cuda(), 30.0)
        k, v = A.paged_kv8_rows(ref[0], ref[2], table, lens), A.paged_kv8_rows(ref[1], ref[3], table, lens)
        ro, bo, _, _ = bounds(q, k, v, lens, 30.0, None)
        check(f"step {step}", out, ro, bo)
    assert same_codes(dev[0], ref[0]) and same_codes(dev[1], ref[1])


def test_decode_and_evict_loop(fa):
    """Decode with weights, evict when the cache is full, go on decoding in the compacted one."""
    g = gen(60)
    b, hq, hkv, d, cap, budget, recent = 2, 8, 2, 64, 48, 24, 6
    k, v = torch.zeros(b, hkv, cap, d, dtype=F16), torch.zeros(b, hkv, cap, d, dtype=F16)
    weight = torch.zeros(b, hkv, cap)
    kc, vc, wc = k.cuda(), v.cuda(), weight.cuda()
    lens = torch.tensor([30, 12])
    k[:], v[:] = randn(g, *k.shape), randn(g, *v.shape)
    kc.copy_(k)
    vc.copy_(v)
    for step in range(60):
        q, nk, nv = randn(g, b, hq, 1, d), randn(g, b, hkv, d), randn(g, b, hkv, d)
        for i in range(b):
            t = int(lens[i])
            for c, x in ((k, nk), (v, nv)):
                c[i, :, t] = x[i]
            kc[i, :, t], vc[i, :, t] = nk[i].cuda(), nv[i].cuda()
            weight[i, :, t] = 0
            wc[i, :, t] = 0
        out, _ = fa.forward_decode_weighted_gqa_fp16(q.cuda(), kc, vc, lens.int().cuda(), wc)
        lens = lens + 1
        ro, bo, p, dp = bounds(q, k, v, lens, 0.0, None)
        check(f"step {step}", out, ro, bo)
        # each step's weights are bounded; the eviction is then checked on the GPU's own sums
        group = p.view(b, hkv, hq // hkv, cap).sum(2)
        assert (wc.cpu().double() - weight.double() - group).abs().max() <= 1e-4
        weight = wc.cpu()
        if int(lens.max()) == cap:
            kc, vc, wc, index, new = fa.evict_by_weight(kc, vc, wc, lens.int().cuda(), budget, recent, cap)
            ref = A.evict_by_weight(k, v, weight, lens, budget, recent, cap)
            for a, r in zip((kc, vc, wc, index, new), ref):
                assert torch.equal(a.cpu(), r)
            k, v, weight, lens = ref[0], ref[1], ref[2], ref[4].long()


def test_streams_and_graphs(fa):
    """The same bits on another stream, from replays with eager calls of other shapes between them (they share
    the workspace pools), and from two captured graphs in turn."""
    g = gen(70)
    q, k, v = randn(g, 4, 16, 1, 128).cuda(), randn(g, 4, 4, 2000, 128).cuda(), randn(g, 4, 4, 2000, 128).cuda()
    lens = torch.tensor([1999, 5, 900, -1], dtype=torch.int32).cuda()
    weight = torch.rand(4, 4, 2000, generator=g).cuda()
    wout = torch.zeros_like(weight)
    codes, scale = make_cache(g, I8, 520, 4, 16, 128)
    codes, scale = codes.cuda(), scale.cuda()
    table = torch.randperm(520, generator=g)[:500].int().view(4, 125).cuda()
    seq = torch.tensor([2000, 6, 901, 0], dtype=torch.int32).cuda()

    def calls():
        o1 = fa.forward_decode_scored_gqa_fp16(q, k, v, lens, 20.0)
        o2, w = fa.forward_decode_weighted_gqa_fp16(q, k, v, lens, weight, wout)
        o3 = fa.forward_paged_decode_kv8_gqa(q, codes, codes, scale, scale, table, seq)
        return [o1, o2, w, o3, *fa.evict_by_weight(k, v, weight, seq, 600, 50, 640)]

    eager = [t.clone() for t in calls()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = calls()
    torch.cuda.current_stream().wait_stream(s)
    for a, e in zip(other, eager):
        assert torch.equal(a, e)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = calls()
        graphs.append((graph, got))
    small = randn(g, 1, 8, 1, 64).cuda(), randn(g, 1, 8, 1500, 64).cuda()
    for _ in range(3):
        for graph, got in graphs:
            for t in got:
                t.zero_()
            fa.forward_decode_scored_gqa_fp16(small[0], small[1], small[1], lens[:1])
            graph.replay()
            torch.cuda.synchronize()
            for a, e in zip(got, eager):
                assert torch.equal(a, e)


def test_refusals(fa):
    q = torch.zeros(2, 4, 1, 64, dtype=F16, device="cuda")
    k = torch.zeros(2, 2, 32, 64, dtype=F16, device="cuda")
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")
    w = torch.zeros(2, 2, 32, device="cuda")
    sl = torch.ones(4, device="cuda")
    codes = torch.zeros(6, 2, 16, 64, dtype=I8, device="cuda")
    sc = torch.ones(6, 2, device="cuda")
    table = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    new = torch.zeros(4, 2, 64, dtype=F16, device="cuda")
    cu = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    dec, wd, pg = fa.forward_decode_scored_gqa_fp16, fa.forward_decode_weighted_gqa_fp16, fa.forward_paged_decode_kv8_gqa
    ap, ev = fa.append_paged_kv8, fa.evict_by_weight
    odd = torch.zeros(6, 2, 24, 64, dtype=I8, device="cuda")
    for i, call in enumerate((
            lambda: dec(q, k, k, lens.long()), lambda: dec(q, k, k, lens[:1]), lambda: dec(q, k, k, lens, -2.0),
            lambda: dec(q, k, k, lens, math.nan), lambda: dec(q, k, k, lens, 0.0, sl[:3]), lambda: dec(q.float(), k.float(), k.float(), lens),
            lambda: dec(q[:, :3].contiguous(), k, k, lens), lambda: dec(q, k, k.transpose(2, 3), lens),
            lambda: dec(q.expand(2, 4, 2, 64).contiguous(), k, k, lens),
            lambda: dec(torch.zeros(2, 4, 1, 264, dtype=F16, device="cuda"), *(torch.zeros(2, 2, 8, 264, dtype=F16, device="cuda"),) * 2, lens),
            lambda: dec(q, k[:, :, :0].contiguous(), k[:, :, :0].contiguous(), lens),
            lambda: wd(q, k, k, lens, w[:, :, :8]), lambda: wd(q, k, k, lens, w.half()), lambda: wd(q, k, k, lens, w, w[:1]),
            lambda: wd(q, k, k, lens, w.cpu()), lambda: wd(q, k, k, lens, w.transpose(0, 1)),
            lambda: pg(q, codes, codes.view(F8), sc, sc, table, lens), lambda: pg(q, odd, odd, sc, sc, table, lens),
            lambda: pg(q, codes, codes, sc[:5], sc, table, lens), lambda: pg(q, codes, codes, sc.half(), sc, table, lens),
            lambda: pg(q, codes, codes, sc, sc, table[:1], lens), lambda: pg(q, codes, codes, sc, sc, table.long(), lens),
            lambda: pg(q, codes, codes, sc, sc, table, lens.long()), lambda: pg(q, codes.view(torch.uint8), codes.view(torch.uint8), sc, sc, table, lens),
            lambda: pg(q, codes[..., :32].contiguous(), codes[..., :32].contiguous(), sc, sc, table, lens),
            lambda: pg(q, codes, codes, sc, sc, table, lens, 1e-9),
            lambda: ap(new, new, cu, lens, 0, codes, codes, sc, sc, table), lambda: ap(new.float(), new, cu, lens, 2, codes, codes, sc, sc, table),
            lambda: ap(new, new, cu[:2], lens, 2, codes, codes, sc, sc, table), lambda: ap(new[:, :1].contiguous(), new[:, :1].contiguous(), cu, lens, 2, codes, codes, sc, sc, table),
            lambda: ap(new, new, cu, lens.long(), 2, codes, codes, sc, sc, table), lambda: ap(new, new, cu, lens, 2, odd, odd, sc, sc, table),
            lambda: ev(k, k, w, lens, 8, 9, 20), lambda: ev(k, k, w, lens, 21, 2, 20), lambda: ev(k, k, w, lens, -1, 0, 20),
            lambda: ev(k, k, w, lens, 8, -1, 20), lambda: ev(k, k, w.half(), lens, 8, 1, 20), lambda: ev(k, k, w, lens.long(), 8, 1, 20),
            lambda: ev(k, k[:1], w, lens, 8, 1, 20), lambda: ev(k, k, w[:, :1], lens, 8, 1, 20), lambda: ev(k.float(), k.float(), w, lens, 8, 1, 20))):
        with pytest.raises(RuntimeError):
            call()
            print("not refused:", i)
