"""The paged serving step as a whole: examples/speculative_decode.py's decoder, with and without drafts."""

from __future__ import annotations

import importlib.util

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu

spec = importlib.util.spec_from_file_location("speculative_decode", ROOT / "examples" / "speculative_decode.py")
example = importlib.util.module_from_spec(spec)
spec.loader.exec_module(example)


def plain_logits(model, ids, slot):
    """Logits of one whole sequence by plain torch in float64, without a cache."""
    f = lambda t: t.double()  # noqa: E731
    h, n = f(model.embed)[ids], len(ids)
    norm = lambda x: x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt()  # noqa: E731
    pos = torch.arange(n, device=model.device)
    for w in model.layers:
        x = norm(h)
        lora = lambda x, i: x @ f(w["a"][i][slot]).T @ f(w["b"][i][slot]).T  # noqa: E731
        q, k, v = (x @ f(m).T + lora(x, i) for i, m in enumerate(w["qkv"].split(model.outs, 0)))
        q, k, v = (t.unflatten(-1, (-1, model.dim)) for t in (q, k, v))
        angle = pos[:, None, None] * model.freqs.double()
        turn = lambda t: torch.cat([t.chunk(2, -1)[0] * angle.cos() - t.chunk(2, -1)[1] * angle.sin(),  # noqa: E731
                                    t.chunk(2, -1)[1] * angle.cos() + t.chunk(2, -1)[0] * angle.sin()], -1)
        group = model.q_heads // model.kv_heads
        s = torch.einsum("thd,jhd->htj", turn(q), turn(k).repeat_interleave(group, 1)) * model.dim ** -0.5
        s = s.masked_fill(pos > pos[:, None], -torch.inf).softmax(-1)
        o = torch.einsum("htj,jhd->thd", s, v.repeat_interleave(group, 1)).flatten(1)
        h = h + o @ f(w["o"]).T + lora(o, 3)
    return norm(h) @ f(model.head).T


PROMPTS = [[3, 1, 4, 1, 5], list(range(90)), [7], [2, 7, 1, 8] * 9]
SLOTS = [0, 3, 1, 2]


@pytest.mark.parametrize("dtype, dim, tol", [(torch.float32, 64, 1e-3), (torch.bfloat16, 64, 0.15),
                                             (torch.float16, 128, 0.03)])
def test_prompts_and_steps_give_the_plain_decoder_s_logits(cuda_dev, dtype, dim, tol):
    """Logits of a ragged prompt batch and of a step of several tokens, against the whole sequence without a cache.
    The logits' standard deviation is about two; the bounds are about ten roundings of their type."""
    model = example.LoRADecoder(hidden=8 * dim, dtype=dtype)
    cache = model.cache(4, 200)
    slots = torch.tensor(SLOTS, dtype=torch.int32, device=cuda_dev)
    seen = [[] for _ in PROMPTS]
    for new in (PROMPTS, [[9, 8, 7], [1], [6, 5, 4, 3], [2]], [[5], [5], [5], [5]]):
        lens = [len(x) for x in new]
        ids = torch.tensor(sum(new, []), device=cuda_dev)
        counts = torch.tensor(lens, dtype=torch.int32, device=cuda_dev)
        got = model.forward(ids, cache, counts, max(lens), slots)
        cache.advance(counts)
        at = 0
        for i, x in enumerate(new):
            seen[i] += x
            want = plain_logits(model, seen[i], SLOTS[i])[-len(x):]
            assert (got[at:at + len(x)].double() - want).abs().max() < tol
            at += len(x)
    cache.check()


def test_greedy_text_does_not_depend_on_the_drafts(cuda_dev):
    """At a low temperature both ways emit the decoder's likeliest tokens, whatever the drafter says; a good drafter
    gets several tokens through in a step."""
    model = example.LoRADecoder(dtype=torch.float32)
    plain, _ = example.generate(model, PROMPTS, SLOTS, 24, 0, None, temperature=1e-4)
    table = torch.randn(model.vocab, model.vocab, device=cuda_dev)
    for row in plain:  # a drafter that knows half of the transitions
        for a, b in list(zip(row, row[1:]))[::2]:
            table[a, b] = 50.0
    drafted, share = example.generate(model, PROMPTS, SLOTS, 24, 3, table, temperature=1e-4)
    for a, b in zip(plain, drafted):
        assert b[:25] == a[:len(b[:25])]
    assert share > 0.1


def test_the_example_runs(cuda_dev, capsys, monkeypatch):
    monkeypatch.setattr("sys.argv", ["speculative_decode.py", "--requests", "3", "--steps", "5"])
    example.main()
    assert "tokens in 5 steps of 3 requests" in capsys.readouterr().out
