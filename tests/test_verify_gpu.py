"""Draft verification against oracle/paged_oracle.py: whole numbers, so every token has to be the oracle's."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from multi_lora_b200 import paged_kv, speculative
from oracle import paged_oracle as O

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def problem(dev, seed, lens, most, vocab, dtype, drafter=True, noise=0.7, keep=0):
    """Target rows, a drafter off by some noise (with ``keep`` > 0 only so many likely tokens), drafts from it."""
    g = torch.Generator(device=dev).manual_seed(seed)
    r, rows = len(lens), sum(n + 1 for n in lens if n >= 0)
    indptr = np.cumsum([0] + [n + 1 for n in lens]).tolist()
    logits = 2 * torch.randn(max(rows, 1), vocab, generator=g, device=dev)
    at = torch.tensor([[min(indptr[i] + j, max(rows, 1) - 1) for j in range(most)] for i in range(r)],
                      dtype=torch.long, device=dev).reshape(r, most)
    guess = logits[at] + noise * torch.randn(r, most, vocab, generator=g, device=dev)
    if keep:
        logits = torch.where(logits >= logits.topk(min(keep, vocab)).values[..., -1:], logits, -torch.inf)
    draft = guess.softmax(-1)
    tokens = torch.multinomial(draft.reshape(r * most, vocab), 1, generator=g).reshape(r, most) if most else at
    target = logits.softmax(-1)
    u = torch.rand(r, most + 1, generator=g, device=dev)
    return dict(target=target.to(DTYPES[dtype]), draft=draft.to(DTYPES[dtype]) if drafter else None, tokens=tokens,
                indptr=torch.tensor(indptr, dtype=torch.int32, device=dev), au=u[:, :most].contiguous(),
                su=u[:, most].contiguous())


def run(pr, status=None):
    out, n = speculative.verify_draft(pr["target"], pr["draft"], pr["tokens"], pr["indptr"], pr["au"], pr["su"],
                                      status=status)
    assert out.dtype == torch.int64 and n.dtype == torch.int32
    return out.cpu().numpy(), n.cpu().numpy()


def want(pr):
    f = lambda t: None if t is None else t.float().cpu().numpy()  # noqa: E731
    return O.verify(f(pr["target"]), f(pr["draft"]), pr["tokens"].cpu().numpy(), pr["indptr"].tolist(),
                    f(pr["au"]), f(pr["su"]))


def check(pr, status=None):
    (a, b), (x, y) = run(pr, status), want(pr)
    assert np.array_equal(b, y) and np.array_equal(a, x)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("drafter", [True, False])
@pytest.mark.parametrize("lens, most, vocab", [
    ([0], 1, 1), ([1], 1, 2), ([3], 3, 1000), ([0, 4, 2, 1], 4, 32000), ([4] * 33, 4, 513), ([2, -1, 0, -1, 3], 3, 4099),
    ([7, 8, 0], 8, 128256), ([0] * 5, 0, 70001),
])
def test_verify_matches_the_oracle(cuda_dev, dtype, drafter, lens, most, vocab):
    for seed in range(4):
        check(problem(cuda_dev, seed, lens, most, vocab, dtype, drafter))


def test_sparse_rows_and_strides(cuda_dev):
    """Rows with a handful of tokens (the rest exactly zero), read out of wider tensors."""
    for seed in range(4):
        pr = problem(cuda_dev, seed, [4, 1, 3, 0], 4, 5003, "f32", keep=6, noise=3.0)
        check(pr)
        for name in ("target", "draft"):
            t = pr[name]
            wide = torch.full((*t.shape[:-1], 5003 + 14), float("nan"), device=cuda_dev)
            wide[..., 3:5006] = t
            pr[name] = wide[..., 3:5006]
        check(pr)


def test_extreme_numbers(cuda_dev):
    """Uniforms at both ends, probabilities of 0, 1, NaN and below 2^-40, equal rows, rows of nothing."""
    v, dev = 300, cuda_dev
    p = torch.zeros(8, v, device=dev)
    p[0, 7] = 1.0
    p[1, 299] = 1.0
    p[2] = 1.0 / v
    p[3, 4], p[3, 5], p[3, 6] = float("nan"), 0.5, 2.0 ** -45
    p[5, 250] = 2.0 ** -41
    p[6, 10], p[6, 11] = 0.25, 0.75
    p[7, 0] = float("inf")
    for u in (0.0, 2.0 ** -24, 0.5, 1 - 2.0 ** -24, 1.0):
        base = dict(target=p, draft=None, tokens=torch.zeros(8, 0, dtype=torch.long, device=dev),
                    indptr=torch.arange(9, dtype=torch.int32, device=dev), au=torch.zeros(8, 0, device=dev),
                    su=torch.full((8,), u, device=dev))
        check(base)
    # equal rows: p - q has no positive part, so a refused draft (u * q >= p only at u = 1) draws from p
    q = p[[2, 6]][:, None].contiguous()
    pr = dict(target=p[[2, 2, 6, 6]].contiguous(), draft=q, tokens=torch.tensor([[9], [11]], device=dev),
              indptr=torch.tensor([0, 2, 4], dtype=torch.int32, device=dev), au=torch.ones(2, 1, device=dev),
              su=torch.tensor([0.3, 0.9], device=dev))
    check(pr)
    assert run(pr)[1].tolist() == [1, 1]
    check(dict(pr, au=torch.zeros(2, 1, device=dev)))  # u = 0 keeps whatever has a probability
    check(dict(pr, draft=torch.zeros_like(q), au=torch.ones(2, 1, device=dev)))  # q(x) = 0: 0 < p keeps


def test_emitted_tokens_follow_the_target(cuda_dev):
    """40000 requests with one draft each over 8 tokens: the first token's frequencies are the target's, within
    five standard deviations of a count."""
    n, v = 40000, 8
    g = torch.Generator(device=cuda_dev).manual_seed(5)
    p = torch.tensor([0.3, 0.05, 0.02, 0.2, 0.03, 0.1, 0.25, 0.05], device=cuda_dev)
    q = torch.tensor([0.1, 0.25, 0.02, 0.1, 0.13, 0.1, 0.05, 0.25], device=cuda_dev)
    drafts = torch.multinomial(q.expand(n, v), 1, generator=g)
    out, _ = speculative.verify_draft(p.expand(2 * n, v).contiguous(), q.expand(n, 1, v).contiguous(), drafts,
                                      torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device=cuda_dev),
                                      torch.rand(n, 1, generator=g, device=cuda_dev),
                                      torch.rand(n, generator=g, device=cuda_dev))
    counts = torch.bincount(out[:, 0], minlength=v).double()
    sigma = (n * p.double() * (1 - p.double())).sqrt()
    assert ((counts - n * p.double()).abs() < 5 * sigma).all()


def test_invalid_rows_and_tokens_are_reported(cuda_dev):
    pr = problem(cuda_dev, 1, [2, 2], 2, 100, "f32")
    status = torch.zeros(1, dtype=torch.int32, device=cuda_dev)
    for bad in ([0, 3, 9], [0, 5, 6], [-2, 1, 4], [4, 0, 3]):
        tokens, n = run(dict(pr, indptr=torch.tensor(bad, dtype=torch.int32, device=cuda_dev)), status)
        assert 0 in n.tolist()
        with pytest.raises(RuntimeError, match="row_indptr"):
            paged_kv.check_status(status)
    for x in (-1, 100, 2 ** 40):
        wrong = pr["tokens"].clone()
        wrong[1, 0] = x
        check(dict(pr, tokens=wrong), status)
        assert run(dict(pr, tokens=wrong))[1][1] == 1
        with pytest.raises(RuntimeError, match="vocabulary"):
            paged_kv.check_status(status)


def test_refusals(cuda_dev):
    pr = problem(cuda_dev, 1, [2, 2], 2, 100, "f32")
    for bad in [dict(target=pr["target"].double()), dict(target=pr["target"].t()), dict(draft=pr["draft"][:, :1]),
                dict(draft=pr["draft"].half()), dict(tokens=pr["tokens"].int()), dict(indptr=pr["indptr"][:2]),
                dict(indptr=pr["indptr"].long()), dict(au=pr["au"][:, :1]), dict(su=pr["su"][:1]),
                dict(su=pr["su"].double()), dict(au=pr["au"].cpu()), dict(target=pr["target"].cpu())]:
        with pytest.raises(RuntimeError):
            run(dict(pr, **bad))


def test_verify_in_a_graph_and_on_another_stream(cuda_dev):
    pr = problem(cuda_dev, 3, [3, 0, 4], 4, 9000, "f32")
    first = run(pr)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, n = speculative.verify_draft(pr["target"], pr["draft"], pr["tokens"], pr["indptr"], pr["au"], pr["su"])
    pr["su"].copy_(1 - pr["su"])
    graph.replay()
    x, y = want(pr)
    assert np.array_equal(out.cpu().numpy(), x) and np.array_equal(n.cpu().numpy(), y)
    pr["su"].copy_(1 - pr["su"])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = run(pr)
    assert all(np.array_equal(a, b) for a, b in zip(again, first))
