"""`logprobs.log_probs` where the logits themselves are large, and of tokens far below the best one.

The tolerances are those of test_logprobs_gpu.py: what they count does not depend on the size of the logits, since every term
begins with an exact (int64) or correctly rounded (float) difference of two of them."""

import pytest
import torch

from test_logprobs_gpu import KINDS, SUM, reference, same

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
