"""Attention with modified scores (tanh cap, distance bias, document and prefix
masks): forward, log-sum-exp and gradients against the 64-bit oracle, at the
sizes and masks where they can go wrong, and the calls that are refused.

Error bounds are worst cases over the roundings the kernels make, element by
element, u = 2^-24 (fp32) and h = 2^-11 (half a step of fp16):
  score     |dy| <= (D + 16) u sum_d |q_d k_d| / sqrt(D) + 8 u (|y| + slope |i - j|)
            (products summed in fp32; the map to the log2 domain, the cap to 4 u, the bias)
  P         |dP| <= P (max |dy| of its row and 2 (N + 16) u for the sum and the exponentials)
  O         |dO| <= (dP + h P + N-key subnormals of unnormalised P) |V| + (N + 16) u P |V| + h |O|
  dS        |d dS| <= dP |dO V^T - delta| + P (D + 16) u (|dO| |V|^T + |dO| |O|) + P |dO| |dO_err|
            + h |dS|, all times the cap's derivative, whose own error is 16 u
  dQ, dK, dV: the products of those with |K|, |Q|, |dO| and the final rounding
where the h terms vanish for fp32.
"""
import math

import pytest
import torch

from oracle import attention as A
from tests.helpers import randn

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32
U = 2.0 ** -24


def gen(seed):
    return torch.Generator().manual_seed(seed)


def slopes_of(h):
    return torch.exp2(-8.0 * torch.arange(1, h + 1, dtype=F32) / h)


def doc_ids_of(b, n, size, g, pad=True):
    """Documents of about `size` tokens; every other row ends in padding, one row starts with it."""
    ids = torch.empty(b, n, dtype=torch.int32)
    for i in range(b):
        at, doc = 0, 5 * i
        while at < n:
            m = int(torch.randint(1, 2 * size, (1,), generator=g))
            ids[i, at:at + m] = doc
            at, doc = at + m, doc + 1
        if pad and i % 2 == 0:
            ids[i, n - max(1, n // 8):] = -1 - i
        if pad and i == 1:
            ids[i, :max(1, n // 5)] = -7
    return ids


def check(what, got, ref, bound):
    got = got.detach().double().cpu()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert bool(torch.isfinite(got).all()), f"{what}: {int((~torch.isfinite(got)).sum())} values are not finite"
    over = (got - ref).abs() - bound
    worst = int(over.argmax())
    assert over.max() <= 0, (f"{what}: {int((over > 0).sum())} of {over.numel()} past the bound; worst {got.flatten()[worst]:.6g} "
                             f"for {ref.flatten()[worst]:.6g}, bound {bound.flatten()[worst]:.3g}")


def run_case(fa, q, k, v, causal, cap, slopes, ids, prefix, dout=None, only_forward=False):
    """Runs forward (and backward) on the GPU and holds them to the bounds; returns the GPU's results."""
    dev = lambda t: None if t is None else t.cuda()
    half = q.dtype == F16
    h_ = 2.0 ** -11 if half else 0.0
    b, hq, n, d = q.shape
    args = (causal, cap, dev(slopes), dev(ids), dev(prefix))
    qc, kc, vc = (t.cuda() for t in (q, k, v))
    if only_forward:
        out, lse = fa.forward_scored(qc, kc, vc, *args), None
    else:
        out, lse = fa.forward_scored_with_lse(qc, kc, vc, *args)
        assert torch.equal(out, fa.forward_scored(qc, kc, vc, *args))
    clean = (lambda t: torch.where((ids < 0)[:, None, :, None], torch.zeros_like(t), t)) if ids is not None else (lambda t: t)
    qd, kd, vd = (clean(t).double() for t in (q, k, v))
    ke, ve = A.expand_kv(kd, hq), A.expand_kv(vd, hq)
    ro, rl, p, y = A.scored(q, k, v, causal, cap, slopes, ids, prefix)
    bt = lambda t: t.transpose(-1, -2)
    i = torch.arange(n).double()
    dist = 0 if slopes is None else slopes.double()[:, None, None] * (i[:, None] - i[None, :]).abs()
    dy = (d + 16) * U * (qd.abs() @ bt(ke.abs())) / math.sqrt(d) + 8 * U * (y.abs() + dist)
    row = torch.where(p > 0, dy, torch.zeros_like(dy)).amax(-1, keepdim=True)
    dp = p * (dy + row + 2 * (n + 16) * U)
    vmax = ve.abs().amax((-2, -1), keepdim=True) if n else 0
    subnormal = n * 2.0 ** -25 * vmax if half else 0.0
    bo = (dp + (h_ + (n + 16) * U) * p) @ ve.abs() + subnormal
    bo = bo * (1 + h_) + (h_ + U) * ro.abs() + (2.0 ** -25 if half else 1e-37)
    check("out", out, ro, bo)
    if lse is not None:
        lse = lse.cpu()
        assert torch.equal(torch.isinf(lse), torch.isinf(rl)), "rows that see nothing"
        fin = torch.isfinite(rl)
        bl = (row[..., 0] + 2 * (n + 16) * U + 8 * U * rl.abs()) + 1e-6
        if fin.any():
            check("lse", lse[fin], rl[fin], bl[fin])
    if dout is None:
        return out
    dq, dk, dv = fa.backward_scored(dout.cuda(), qc, kc, vc, out, lse.cuda(), *args)
    rq, rk, rv = A.scored_backward(dout, q, k, v, causal, cap, slopes, ids, prefix)
    do = clean(dout).double()
    dov = do @ bt(ve)
    delta = (do * ro).sum(-1, keepdim=True)
    dyg = p * (dov - delta)
    cap_d = 1.0
    if cap:
        t = (qd @ bt(ke)) / math.sqrt(d) / cap
        cap_d = 1 - torch.tanh(t) ** 2
    ds = dyg * cap_d
    bds = dp * (dov - delta).abs() + p * (d + 16) * U * (do.abs() @ bt(ve.abs()) + (do.abs() * ro.abs()).sum(-1, keepdim=True))
    bds = bds + p * (do.abs() * bo).sum(-1, keepdim=True)
    bds = bds * cap_d + 16 * U * dyg.abs() + h_ * (ds.abs() + bds) + (2.0 ** -25 * (p > 0) if half else 0.0)
    group = lambda t: t.view(b, k.shape[1], hq // k.shape[1], n, d).sum(2)
    acc = (n * hq // k.shape[1] + 16) * U
    scale = 1 / math.sqrt(d)
    tiny = 2.0 ** -24 if half else 1e-37
    for what, got, ref, bound in (
            ("dq", dq, rq, scale * ((bds + acc * ds.abs()) @ ke.abs())),
            ("dk", dk, rk, scale * group(bt(bds + acc * ds.abs()) @ qd.abs())),
            ("dv", dv, rv, group(bt(dp + (h_ + acc) * p + (2.0 ** -25 * (p > 0) if half else 0.0)) @ do.abs()))):
        check(what, got, ref, bound * (1 + h_) + (h_ + U) * ref.abs() + tiny)
    return out, lse.cuda(), dq, dk, dv


def make(seed, dtype, b, hq, hkv, n, d, scale=1.0):
    g = gen(seed)
    q = (randn(g, b, hq, n, d, dtype=F32) * scale).to(dtype)
    k, v = randn(g, b, hkv, n, d, dtype=dtype), randn(g, b, hkv, n, d, dtype=dtype)
    return g, q, k, v, randn(g, b, hq, n, d, dtype=dtype)


#         b hq hkv n    d
SHAPES = [(1, 1, 1, 1, 64), (2, 2, 1, 2, 8), (1, 4, 2, 31, 64), (2, 4, 4, 33, 80), (1, 6, 2, 65, 128), (2, 3, 3, 129, 36),
          (3, 4, 1, 200, 96), (1, 8, 2, 300, 128), (2, 2, 2, 513, 64), (1, 2, 1, 257, 120)]
MODS = {"plain": (0.0, False, 0, False), "cap": (5.0, False, 0, False), "bias": (0.0, True, 0, False),
        "docs": (0.0, False, 40, False), "prefix": (0.0, False, 0, True), "cap_docs": (50.0, False, 90, False),
        "bias_docs_prefix": (0.0, True, 60, True), "all": (2.0, True, 25, True)}


@pytest.mark.parametrize("mods", list(MODS))
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("b,hq,hkv,n,d", SHAPES)
def test_forward_and_gradients(fa, dtype, b, hq, hkv, n, d, causal, mods):
    cap, bias, docs, pre = MODS[mods]
    if pre and not causal:
        pytest.skip("a prefix needs a causal mask")
    g, q, k, v, do = make(n * 7 + d, dtype, b, hq, hkv, n, d, scale=3.0)
    ids = doc_ids_of(b, n, docs, g) if docs else None
    prefix = torch.randint(0, n + 2, (b,), generator=g, dtype=torch.int32) if pre else None
    run_case(fa, q, k, v, causal, cap, slopes_of(hq) if bias else None, ids, prefix, do)


@pytest.mark.parametrize("d", [136, 192, 200, 250, 256])
@pytest.mark.parametrize("mods", ["cap", "bias", "docs", "all"])
def test_wide_heads_forward(fa, d, mods):
    cap, bias, docs, pre = MODS[mods]
    g, q, k, v, _ = make(d, F16, 2, 4, 2, 150, d)
    ids = doc_ids_of(2, 150, docs, g) if docs else None
    run_case(fa, q, k, v, True, cap, slopes_of(4) if bias else None, ids,
             torch.tensor([3, 90], dtype=torch.int32) if pre else None, only_forward=True)


@pytest.mark.parametrize("b,hq,hkv,n,d,dtype", [
    (8, 32, 8, 300, 64, F16), (5, 8, 8, 640, 128, F16), (1, 64, 8, 1100, 128, F16), (3, 12, 4, 420, 96, F16),
    (9, 8, 8, 300, 64, F32), (2, 16, 16, 400, 128, F32), (40, 8, 8, 70, 64, F32)])
@pytest.mark.parametrize("mods", ["cap_docs", "bias_docs_prefix", "plain"])
def test_grids(fa, b, hq, hkv, n, d, dtype, mods):
    """Grids of whole and split blocks, units that fill the XCDs evenly and not, short last rounds: every
    head and row is written, equal for equal inputs: the batch's first row is repeated in its last."""
    cap, bias, docs, pre = MODS[mods]
    g, q, k, v, do = make(b + n, dtype, b, hq, hkv, n, d)
    ids = doc_ids_of(b, n, docs, g) if docs else None
    prefix = torch.randint(0, n + 1, (b,), generator=g, dtype=torch.int32) if pre else None
    for t in (q, k, v, do, ids, prefix):
        if t is not None:
            t[-1] = t[0]
    dev = lambda t: None if t is None else t.cuda()
    args = (True, cap, dev(slopes_of(hq)) if bias else None, dev(ids), dev(prefix))
    out, lse = fa.forward_scored_with_lse(q.cuda(), k.cuda(), v.cuda(), *args)
    grads = fa.backward_scored(do.cuda(), q.cuda(), k.cuda(), v.cuda(), out, lse, *args)
    for t in (out, lse, *grads):
        assert torch.equal(t[0], t[-1])
    i = b // 2
    cut = lambda t: None if t is None else t[i:i + 1]
    ref = run_case(fa, cut(q), cut(k), cut(v), True, cap, slopes_of(hq) if bias else None, cut(ids), cut(prefix), cut(do))
    # the single row may be split otherwise than the batch: equal to the sum's order
    for a, r in zip((out, lse, *grads), ref):
        a, r = a[i:i + 1].float(), r.float()
        fin = torch.isfinite(r)
        assert torch.equal(torch.isfinite(a), fin)
        tol = (2e-3 if dtype == F16 else 2e-5) * max(1.0, float(r[fin].abs().max()))
        assert (a[fin] - r[fin]).abs().max() <= tol


@pytest.mark.parametrize("n,size", [(2300, 30), (4500, 700), (4500, 5000)])
def test_long_rows_walk_only_their_documents(fa, n, size):
    """Rows past one group of 64 sub-tiles, documents that come back later in the row, ids in no order."""
    g, q, k, v, do = make(n, F16, 1, 1, 1, n, 64)
    ids = doc_ids_of(1, n, size, g)
    perm = torch.randperm(int(ids.max()) + 1, generator=g).to(torch.int32)
    ids = torch.where(ids >= 0, perm[ids.clamp(min=0).long()], ids)
    ids[0, 17:40] = ids[0, n // 2]
    ids[0, n - 70:n - 60] = ids[0, 3]
    for causal in (True, False):
        run_case(fa, q, k, v, causal, 30.0, None, ids, None, do)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d", [64, 128, 20])
def test_padding_may_hold_anything(fa, dtype, d):
    """NaN and infinities in rows of negative id reach nothing, and their own results are zeros."""
    b, hq, hkv, n = 2, 4, 2, 150
    g, q, k, v, do = make(5 + d, dtype, b, hq, hkv, n, d)
    ids = doc_ids_of(b, n, 30, g)
    ids[0, 40:47] = -1
    bad = torch.tensor([math.nan, math.inf, -math.inf], dtype=dtype)
    for i in range(b):
        pad = (ids[i] < 0).nonzero()[:, 0]
        for t in (q, k, v, do):
            t[i][:, pad] = bad[torch.randint(0, 3, t[i][:, pad].shape, generator=g)]
    for causal in (True, False):
        out, lse, dq, dk, dv = run_case(fa, q, k, v, causal, 4.0, None, ids, None, do)
        for i in range(b):
            pad = (ids[i] < 0).nonzero()[:, 0].cuda()
            for t in (out, dq, dk, dv):
                assert not t[i][:, pad].any()


def test_all_rows_padding(fa):
    g, q, k, v, do = make(3, F16, 2, 2, 2, 70, 64)
    ids = torch.full((2, 70), -1, dtype=torch.int32)
    ids[1, 5] = 2
    out, lse, dq, dk, dv = run_case(fa, q, k, v, False, 0.0, None, ids, None, do)
    assert torch.isinf(lse[0]).all() and not out[0].any() and not dv[0].any()
    assert torch.equal(out[1, :, 5], v.cuda()[1, :, 5])


@pytest.mark.parametrize("scale", [1.0, 30.0, 3000.0])
def test_cap_over_its_whole_range(fa, scale):
    """Scores far below, about and far past the cap (both forms of the tanh in one tile)."""
    for dtype in (F16, F32):
        g, q, k, v, do = make(int(scale), dtype, 1, 2, 2, 100, 64)
        q = (q.float() * torch.exp(torch.randn(100, 1, generator=g)) * scale / 30).to(dtype)
        run_case(fa, q, k, v, True, 20.0, None, None, None, do)


def test_steep_and_zero_slopes(fa):
    g, q, k, v, do = make(9, F32, 1, 4, 4, 700, 64)
    run_case(fa, q, k, v, True, 0.0, torch.tensor([0.0, 40.0, 1e-4, 3.0]), None, None, do)
    run_case(fa, q, k, v, False, 0.0, torch.tensor([0.0, 40.0, -0.01, 3.0]), None, None, do)


def test_prefix_edges(fa):
    for n in (64, 130):
        g, q, k, v, do = make(n, F16, 6, 2, 1, n, 64)
        prefix = torch.tensor([0, 1, n, n + 50, -3, 33], dtype=torch.int32)
        run_case(fa, q, k, v, True, 0.0, None, None, prefix, do)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("mods", ["cap", "all"])
def test_gradients_against_differences(fa, dtype, mods):
    """sum(out * dout) along a direction, by central differences of the 64-bit forward, against the kernels'
    gradients; what the difference itself is off by (third order) is measured from a step of half the size."""
    cap, bias, docs, pre = MODS[mods]
    b, hq, hkv, n, d = 1, 4, 2, 90, 64
    g, q, k, v, do = make(77, dtype, b, hq, hkv, n, d)
    ids = doc_ids_of(b, n, docs, g) if docs else None
    prefix = torch.tensor([20], dtype=torch.int32) if pre else None
    slopes = slopes_of(hq) if bias else None
    _, _, dq, dk, dv = run_case(fa, q, k, v, True, cap, slopes, ids, prefix, do)
    live = torch.ones(b, 1, n, 1) if ids is None else (ids >= 0).double()[:, None, :, None]
    f = lambda *t: float((A.scored(*t, True, cap, slopes, ids, prefix)[0] * do.double() * live).sum())
    for i, (x, grad) in enumerate(((q, dq), (k, dk), (v, dv))):
        way = torch.randn(x.shape, generator=g, dtype=torch.float64)
        def diff(step):
            hi, lo = ([t.double() for t in (q, k, v)] for _ in range(2))
            hi[i], lo[i] = hi[i] + step * way, lo[i] - step * way
            return (f(*hi) - f(*lo)) / (2 * step)
        a, c = diff(1e-4), diff(5e-5)
        along = float((grad.double().cpu() * way).sum())
        # rounding of the gradient's elements: independent signs against a random direction, six deviations
        rounding = 6 * (2.0 ** -9 if dtype == F16 else 1e-5) * float((grad.double().cpu() * way).norm())
        assert abs(along - c) <= rounding + 4 * abs(a - c) + 1e-6, (i, along, c)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_autograd_streams_and_graph(fa, dtype):
    """The autograd wrapper's gradients, shared KV heads and non-contiguous inputs among them; the same bits on
    another stream and from every replay of a captured graph."""
    from flash_attn_autograd import flash_attn_scored

    g, q, k, v, do = make(21, dtype, 2, 8, 2, 260, 64)
    ids = doc_ids_of(2, 260, 50, g).cuda()
    slopes = slopes_of(8).cuda()
    args = (True, 30.0, slopes, ids, torch.tensor([10, 0], dtype=torch.int32).cuda())
    qc, kc, vc, dc = (t.cuda() for t in (q, k, v, do))
    out, lse = fa.forward_scored_with_lse(qc, kc, vc, *args)
    eager = fa.backward_scored(dc, qc, kc, vc, out, lse, *args)
    # a [B, N, H, D] tensor seen as [B, H, N, D]
    leaves = [t.transpose(1, 2).contiguous().requires_grad_() for t in (qc, kc, vc)]
    o = flash_attn_scored(*(t.transpose(1, 2) for t in leaves), *args)
    o.backward(dc.transpose(1, 2).contiguous().transpose(1, 2))
    assert torch.equal(o, out)
    for t, e in zip(leaves, eager):
        assert torch.equal(t.grad.transpose(1, 2), e)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        on_s = fa.backward_scored(dc, qc, kc, vc, *fa.forward_scored_with_lse(qc, kc, vc, *args), *args)
    torch.cuda.current_stream().wait_stream(s)
    for a, e in zip(on_s, eager):
        assert torch.equal(a, e)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o2, l2 = fa.forward_scored_with_lse(qc, kc, vc, *args)
        captured = fa.backward_scored(dc, qc, kc, vc, o2, l2, *args)
    for _ in range(3):
        for t in (o2, l2, *captured):
            t.zero_()
        fa.backward_scored(dc, qc, kc, vc, out, lse, *args)
        graph.replay()
        torch.cuda.synchronize()
        for a, e in zip((o2, l2, *captured), (out, lse, *eager)):
            assert torch.equal(a, e)


def test_unaligned_storage(fa):
    """Tensors that start two bytes past a 16-byte boundary."""
    g, q, k, v, do = make(31, F16, 1, 4, 2, 100, 64)
    shift = lambda t: torch.cat([torch.zeros(1, dtype=t.dtype), t.flatten()]).cuda()[1:].view(t.shape)
    ids = doc_ids_of(1, 100, 30, g)
    args = (True, 8.0, slopes_of(4).cuda(), ids.cuda(), None)
    qs, ks, vs, ds = (shift(t) for t in (q, k, v, do))
    assert qs.data_ptr() % 16 == 2
    run_case(fa, q, k, v, True, 8.0, slopes_of(4), ids, None, do)
    out, lse = fa.forward_scored_with_lse(qs, ks, vs, *args)
    grads = fa.backward_scored(ds, qs, ks, vs, out, lse, *args)
    o2, l2 = fa.forward_scored_with_lse(*(t.cuda() for t in (q, k, v)), *args)
    g2 = fa.backward_scored(do.cuda(), *(t.cuda() for t in (q, k, v)), o2, l2, *args)
    for a, r in zip((out, *grads), (o2, *g2)):
        assert (a.float() - r.float()).abs().max() <= 2 ** -9 * r.float().abs().max()


def test_empty(fa):
    for shape in ((0, 4, 5, 64), (2, 4, 0, 64)):
        q = torch.zeros(shape, dtype=F16, device="cuda")
        k = torch.zeros((shape[0], 2) + shape[2:], dtype=F16, device="cuda")
        out, lse = fa.forward_scored_with_lse(q, k, k, True, 3.0)
        assert out.shape == q.shape and lse.shape == shape[:3]
        dq, dk, dv = fa.backward_scored(q, q, k, k, out, lse, True, 3.0)
        assert dq.shape == q.shape and dk.shape == k.shape


def test_refusals(fa):
    from flash_attn_autograd import flash_attn_scored

    q = torch.zeros(2, 4, 16, 64, dtype=F16, device="cuda")
    k = torch.zeros(2, 2, 16, 64, dtype=F16, device="cuda")
    ids = torch.zeros(2, 16, dtype=torch.int32, device="cuda")
    pre = torch.zeros(2, dtype=torch.int32, device="cuda")
    sl = torch.ones(4, device="cuda")
    wide = torch.zeros(2, 4, 16, 136, dtype=F16, device="cuda")
    f32wide = wide.float()
    for call in (
            lambda: fa.forward_scored(q, k, k, True, -1.0), lambda: fa.forward_scored(q, k, k, True, math.nan),
            lambda: fa.forward_scored(q, k, k, True, math.inf), lambda: fa.forward_scored(q, k, k, True, 1e-5),
            lambda: fa.forward_scored(q, k, k, False, 0.0, None, None, pre),
            lambda: fa.forward_scored(q, k, k, True, 0.0, sl[:2]), lambda: fa.forward_scored(q, k, k, True, 0.0, sl.double()),
            lambda: fa.forward_scored(q, k, k, True, 0.0, sl.cpu()), lambda: fa.forward_scored(q, k, k, True, 0.0, None, ids.long()),
            lambda: fa.forward_scored(q, k, k, True, 0.0, None, ids[:, :8]),
            lambda: fa.forward_scored(q, k, k, True, 0.0, None, ids.t().contiguous().t()),
            lambda: fa.forward_scored(q, k, k, True, 0.0, None, None, pre[:1]),
            lambda: fa.forward_scored(q.transpose(1, 2), k, k, True), lambda: fa.forward_scored(q, k.float(), k, True),
            lambda: fa.forward_scored(q, k[:, :, :8].contiguous(), k, True), lambda: fa.forward_scored(q.double(), k.double(), k.double(), True),
            lambda: fa.forward_scored(q[:, :3].contiguous(), k, k, True), lambda: fa.forward_scored(q.cpu(), k.cpu(), k.cpu(), True),
            lambda: fa.forward_scored_with_lse(wide, wide, wide, True), lambda: fa.forward_scored(f32wide, f32wide, f32wide, True),
            lambda: fa.backward_scored(q, q, k, k, q, torch.zeros(2, 4, 15, device="cuda"), True),
            lambda: fa.backward_scored(q[:1], q, k, k, q, torch.zeros(2, 4, 16, device="cuda"), True),
            lambda: flash_attn_scored(q, k, k, True, 0.0, sl.clone().requires_grad_())):
        with pytest.raises(RuntimeError):
            call()
