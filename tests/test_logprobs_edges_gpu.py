"""`logprobs.log_probs` where the logits themselves are large, and of tokens far below the best one.

The tolerances are those of test_logprobs_gpu.py: what they count does not depend on the size of the logits, since every term
begins with an exact (int64) or correctly rounded (float) difference of two of them."""

import pytest
import torch

from test_logprobs_gpu import FR, SUM, reference, same

pytestmark = pytest.mark.gpu
SIZES = (1e3, 4e3, 1e5, 1e6, 1.5e7, 1e8, 1e9, 1e10, 1e20, 1e30, 1e37)


@pytest.mark.parametrize("kind", ("float32", "bfloat16"))
@pytest.mark.parametrize("V", [1024, 5000, 130000])
@pytest.mark.parametrize("sign", [1, -1])
def test_logits_of_any_size(sign, V, kind):
    """Constant rows, and rows of entries around a common offset: 3 apart, or some units in the last place where that is more."""
    from bitexact_llm_b200.logprobs import log_probs
    T = getattr(torch, kind)
    g = torch.Generator().manual_seed(V)
    rows, tok = [], []
    for size in SIZES:
        unit = size * torch.finfo(T).eps
        rows.append(torch.full((V,), sign * size).to(T))
        rows.append((sign * size + torch.randn(V, generator=g, dtype=torch.float64) * max(3.0, 2 * unit)).to(T))
        tok += [V // 2, int(torch.randint(V, (1,), generator=g))]
    x, tok = torch.stack(rows), torch.tensor(tok)
    same(log_probs(x.cuda(), tok.cuda(), 5), reference(x, tok, 5), V)


@pytest.mark.parametrize("kind", ("float32", "bfloat16"))
def test_logits_that_grow_along_the_row(kind):
    """A thread's reference passes every size, up and down."""
    from bitexact_llm_b200.logprobs import log_probs
    T, V = getattr(torch, kind), 40000
    up = torch.logspace(-2, 12, V, dtype=torch.float64)
    x = torch.stack([up, up.flip(0), -up, -up.flip(0)]).to(T)
    tok = torch.tensor([V - 1, 0, 0, V - 1])
    same(log_probs(x.cuda(), tok.cuda(), 3), reference(x, tok, 3), V)


@pytest.mark.parametrize("fr", [0, 8, 16, 24, 30, 40])
@pytest.mark.parametrize("V", [6, 3000, 70000])
def test_fixed_point_tokens_far_below_the_best(V, fr):
    """Their log probability is their distance, whatever e^ of it is; at every binary point the same."""
    from bitexact_llm_b200.logprobs import MASKED, log_probs
    far = [0, -255, -257, -1000, -10 ** 5, -10 ** 6]
    x = torch.full((len(far) + 1, V), MASKED, dtype=torch.long)
    for i in range(len(far)):
        x[i, :6] = torch.tensor(far) << fr
        x[i, 1] += i
    x[-1] = -(torch.arange(V) % 3000 << fr)
    tok = torch.tensor([*range(6), min(V - 1, 2999)])
    same(log_probs(x.cuda(), tok.cuda(), 6, fr=fr), reference(x, tok, 6, fr), V)


def test_fixed_point_tokens_at_the_ends_of_the_type():
    from bitexact_llm_b200.logprobs import MASKED, log_probs
    low, high = MASKED + 1, (1 << 63) - 1
    x = torch.full((2, 700), MASKED, dtype=torch.long)
    x[:, 3], x[:, 5], x[:, 600] = high, low, 0
    r = log_probs(x.cuda(), torch.tensor([5, 7]).cuda(), 4)
    want = torch.tensor([0.0, -high * 2.0 ** -FR, (low - high) * 2.0 ** -FR], dtype=torch.float64)
    # token 7 is masked: behind the three others and the masked tokens 0, 1, 2, 4 and 6
    assert r.top_ids.tolist() == [[3, 600, 5, -1]] * 2 and r.rank.tolist() == [3, 1 + 3 + 5]
    assert ((r.top_logp[:, :3].double().cpu() - want).abs() <= SUM + 2.0 ** -22 * want.abs()).all() and (r.top_logp[:, 3] == -torch.inf).all()
    assert r.logp[0] == r.top_logp[0, 2] and r.logp[1] == -torch.inf
