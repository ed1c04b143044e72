"""The 64-bit oracle of attention with modified scores against loops over its
definition, its gradients against differences, and the module's checks of
arguments that need no GPU."""
import math

import pytest
import torch

from oracle import attention as A


def loops(q, k, v, causal, cap, slopes, ids, prefix):
    b_, hq, n, d = q.shape
    out, lse = torch.zeros(b_, hq, n, d, dtype=torch.float64), torch.full((b_, hq, n), -math.inf, dtype=torch.float64)
    for b in range(b_):
        for h in range(hq):
            kh = h // (hq // k.shape[1])
            for i in range(n):
                seen = {}
                for j in range(n):
                    if ids is not None and (int(ids[b, i]) != int(ids[b, j]) or int(ids[b, i]) < 0):
                        continue
                    if causal and j > i and not (prefix is not None and j < int(prefix[b])):
                        continue
                    s = sum(float(x) * float(y) for x, y in zip(q[b, h, i], k[b, kh, j])) / math.sqrt(d)
                    s = cap * math.tanh(s / cap) if cap else s
                    seen[j] = s - (float(slopes[h]) * abs(i - j) if slopes is not None else 0.0)
                if seen:
                    top = max(seen.values())
                    total = sum(math.exp(s - top) for s in seen.values())
                    lse[b, h, i] = top + math.log(total)
                    out[b, h, i] = sum(math.exp(s - top) / total * v[b, kh, j].double() for j, s in seen.items())
    return out, lse


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("cap,bias,docs,pre", [(0.0, False, False, False), (1.5, True, False, True),
                                               (0.7, False, True, False), (0.0, True, True, True)])
def test_oracle(causal, cap, bias, docs, pre):
    if pre and not causal:
        pytest.skip("a prefix needs a causal mask")
    g = torch.Generator().manual_seed(3)
    q = torch.randn(2, 4, 7, 5, generator=g)
    k, v = (torch.randn(2, 2, 7, 5, generator=g) for _ in range(2))
    slopes = torch.tensor([0.0, 0.5, 1.0, -0.25]) if bias else None
    ids = torch.tensor([[3, 3, 1, 1, 1, 3, -1], [-1, 0, 0, 9, 9, 9, 9]], dtype=torch.int32) if docs else None
    prefix = torch.tensor([4, 0], dtype=torch.int32) if pre else None
    args = (causal, cap, slopes, ids, prefix)
    out, lse = A.scored(q, k, v, *args)[:2]
    ro, rl = loops(q, k, v, *args)
    assert torch.allclose(out, ro, atol=1e-12) and torch.allclose(lse, rl, atol=1e-12)
    do = torch.randn(q.shape, generator=g).double()
    grads = A.scored_backward(do, q, k, v, *args)
    live = 1.0 if ids is None else (ids >= 0).double()[:, None, :, None]
    for i, x in enumerate((q, k, v)):
        way = torch.randn(x.shape, generator=g).double()
        f = lambda step: float((A.scored(*(t.double() + (step * way if j == i else 0) for j, t in enumerate((q, k, v))),
                                         *args)[0] * do * live).sum())
        assert abs((f(1e-5) - f(-1e-5)) / 2e-5 - float((grads[i] * way).sum())) < 1e-7
