"""Attention with modified scores and the 8-bit cache at values and orders that their other tests do not reach:
document ids at the ends of int32, every fp16 value through the append's rounding, calls on two streams at once,
training through autograd in a captured graph, and weights summed into an array of their own beside the first."""
import pytest
import torch

from oracle import attention as A
from tests.helpers import randn

pytestmark = pytest.mark.gpu
F16, F32, I8, F8 = torch.float16, torch.float32, torch.int8, torch.float8_e4m3fn
TOP = 2 ** 31 - 1


def gen(seed):
    return torch.Generator().manual_seed(seed)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("causal", [True, False])
def test_ids_at_the_ends_of_int32(fa, dtype, causal):
    """Only which ids are equal and which are negative matters: the same bits from small ids and from extreme ones."""
    g = gen(1)
    n = 300
    small = torch.full((2, n), -1, dtype=torch.int32)
    small[0, 10:150], small[0, 150:290] = 0, 1
    small[1, :40], small[1, 70:200], small[1, 200:] = 0, 1, 2
    far = torch.where(small < 0, torch.tensor(-TOP - 1), torch.tensor([0, TOP - 1, TOP])[small.clamp(min=0).long()])
    far[0, :10], far[0, 150:290] = -TOP + 1, TOP
    q, do = (randn(g, 2, 4, n, 64, dtype=dtype).cuda() for _ in range(2))
    k, v = (randn(g, 2, 2, n, 64, dtype=dtype).cuda() for _ in range(2))

    def run(ids):
        args = (causal, 5.0, None, ids.int().cuda(), None)
        out, lse = fa.forward_scored_with_lse(q, k, v, *args)
        return (out, lse, *fa.backward_scored(do, q, k, v, out, lse, *args))

    for a, b in zip(run(small), run(far)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [I8, F8])
@pytest.mark.parametrize("d", [64, 40])
def test_append_rounds_every_value(fa, dtype, d):
    """Every finite fp16 value under page maxima of many sizes (its neighbours in the page no greater): the codes of
    the quotient correctly rounded in fp32, exactly."""
    g = gen(2)
    values = torch.arange(0x7c00, dtype=torch.int32).to(torch.int16).view(F16)
    tops = torch.cat([values[[1, 2, 3, 127, 1023, 1024, 1025, 0x3c00, 0x3c01, 0x7bff]],
                      values[torch.randint(1, 0x7c00, (40,), generator=g)]])
    rows, page = 16, 16
    pages = []
    for top in tops:
        fit = values[values <= top]
        x = fit[torch.randint(0, len(fit), (rows * d,), generator=g)]
        x = torch.where(torch.rand(rows * d, generator=g) < 0.5, -x, x)
        x[0] = top
        pages.append(x.view(rows, 1, d))
    # and all values at once, under the greatest
    whole = torch.cat([values, -values, torch.zeros(-2 * len(values) % (rows * d - 1), dtype=F16)]).view(-1, rows * d - 1)
    whole = torch.cat([torch.full((len(whole), 1), float(values[-1]), dtype=F16), whole], 1)
    k = torch.cat(pages + [whole.view(-1, 1, d)])
    count = k.shape[0] // page
    cu, lens = torch.tensor([0, k.shape[0]]), torch.tensor([0])
    table = torch.randperm(count, generator=g).int()[None]
    cache = torch.zeros(count, 1, page, d, dtype=I8).view(dtype)
    scale = torch.zeros(count, 1)
    ref = A.append_paged_kv8(k, -k, cu, lens, k.shape[0], cache, cache, scale, scale, table)
    got = [t.clone().cuda() for t in (cache, cache, scale, scale)]
    fa.append_paged_kv8(k.cuda(), (-k).cuda(), cu.int().cuda(), lens.int().cuda(), k.shape[0], *got, table.cuda())
    for a, r in zip(got, ref):
        assert torch.equal(a.cpu().view(torch.uint8), r.view(torch.uint8))


def test_two_streams_at_once(fa):
    """Calls in flight on two streams share no workspace: each gives its own eager bits."""
    g = gen(3)
    q, k, v = (randn(g, 4, h, n, 128).cuda() for h, n in ((16, 1), (4, 3001), (4, 3001)))
    lens = torch.tensor([3000, 17, 1400, 2999], dtype=torch.int32).cuda()
    x, y, z, do = (randn(g, 2, h, 700, 64).cuda() for h in (8, 2, 2, 8))
    ids = (torch.arange(700, dtype=torch.int32) // 90).expand(2, 700).contiguous().cuda()
    weight = torch.rand(4, 4, 3001, generator=g).cuda()

    def calls():
        out, lse = fa.forward_scored_with_lse(x, y, z, True, 20.0, None, ids)
        o1 = fa.forward_decode_scored_gqa_fp16(q, k, v, lens, 20.0)
        o2, w = fa.forward_decode_weighted_gqa_fp16(q, k, v, lens, weight, weight.clone())
        return [out, lse, *fa.backward_scored(do, x, y, z, out, lse, True, 20.0, None, ids), o1, o2, w]

    eager = calls()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(calls())
    torch.cuda.synchronize()
    for call in got:
        for a, e in zip(call, eager):
            assert torch.equal(a, e)


def test_training_step_in_a_graph(fa):
    """flash_attn_scored's forward and backward captured through autograd; replays on new inputs give the eager bits."""
    from flash_attn_autograd import flash_attn_scored

    g = gen(4)
    data = [[randn(g, 1, h, 200, 64).cuda() for h in (4, 2, 2, 4)] for _ in range(3)]
    slopes = torch.tensor([0.5, 0.25, 0.125, 0.0625]).cuda()

    def step(q, k, v, do):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = flash_attn_scored(*leaves, True, 30.0, slopes)
        return [out.detach(), *torch.autograd.grad(out, leaves, do)]

    eager = [[t.clone() for t in step(*d)] for d in data]
    static = [t.clone() for t in data[0]]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(*static)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*static)
    for d, e in list(zip(data, eager)) * 2:
        for t, x in zip(static, d):
            t.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        for a, r in zip(got, e):
            assert torch.equal(a, r)


def test_weights_beside_each_other(fa):
    """weight and weight_out may be one array or two apart, neighbours included; two that overlap in part are refused."""
    g = gen(5)
    q, k, v = (randn(g, 2, h, n, 64).cuda() for h, n in ((4, 1), (2, 50), (2, 50)))
    lens = torch.tensor([49, 20], dtype=torch.int32).cuda()
    pool = torch.rand(3 * 200, generator=g).cuda()
    at = lambda i: pool[i:i + 200].view(2, 2, 50)
    first = at(0).clone()
    _, want = fa.forward_decode_weighted_gqa_fp16(q, k, v, lens, first, torch.zeros_like(first))
    before = at(200).clone()
    _, got = fa.forward_decode_weighted_gqa_fp16(q, k, v, lens, at(0), at(200))
    live = torch.arange(50)[None, None, :] <= lens.cpu()[:, None, None]
    assert torch.equal(got.cpu(), torch.where(live, want.cpu(), before.cpu())) and torch.equal(at(0), first)
    for shift in (4, 100, 196):
        with pytest.raises(RuntimeError):
            fa.forward_decode_weighted_gqa_fp16(q, k, v, lens, at(0), at(shift))
