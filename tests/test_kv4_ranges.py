"""Attention over the 4-bit cache at the ends of the numbers' range, against 64 bits (tests/kv4_reference.py), in the kernel
for few rows and in the one for prompts. Tolerances: tests/test_kv4.py's (which covers the prompts', tests/test_kv4_prompts.py),
whose slack is a channel's own largest value, so that quiet channels are not measured against loud ones."""

import pytest
import torch

from tests import kv4_reference as ref
from tests.test_kv4 import _attend, _bf16, _check

pytestmark = pytest.mark.gpu

# lens, new tokens, query heads, KV heads: two tokens of a decode step, and 32 blocks of a prompt
FEW, PROMPT = ([200, 40], None, 4, 2), ([150], [150], 32, 16)


@pytest.mark.parametrize("lens,news,hq,hkv", [FEW, PROMPT])
@pytest.mark.parametrize("power", [-133, -126, -120, -113, 100, 120])
def test_queries_at_the_ends_of_the_range(sk, lens, news, hq, hkv, power):
    """Queries of up to 127 x 2^power (at -133: below the normal numbers) with a scale that makes the scores ordinary. The scores'
    error bound scales with |scale q|, whose mean is 0.8 d^-1/2 here as there."""
    g = torch.Generator().manual_seed(power + 200)
    rows = len(lens) if news is None else sum(news)
    n = (40 * torch.randn(rows, hq, 128, generator=g)).round().clamp(-127, 127)
    q = (n.double() * 2.0 ** power).to(torch.bfloat16)
    assert torch.equal(q.double(), n.double() * 2.0 ** power)
    got, want, slack = _attend(sk, g, lens, news, 16, hq, hkv, 128, 64, scale=2.0 ** -power / 40 * 128 ** -0.5, q=q)
    _check(got, want, slack, f"2^{power}")
