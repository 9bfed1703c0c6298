"""Rows of many keys whose weights are small against one: the sum over them is the lse's, and does not stand still at its largest
item."""
import math

import pytest
import torch

import attention_oracle as oracle
from gpu_util import log

pytestmark = pytest.mark.gpu

DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16}


@pytest.mark.parametrize("suffix", ["bf16", "f16"])
@pytest.mark.parametrize("above", [15.0, 17.0, 19.0])
@pytest.mark.parametrize("rows,how", [(1, "one part"), (1, "parts"), (60, "one part"), (60, "parts"), (1, "packed"), (130, "packed")])
def test_sum_over_many_small_weights(hip, dev, suffix, above, rows, how):
    """100,000 keys of which the first scores `above` more than about all others.  A lane adds the sums of at least 16 of its
    keys to its total, so 100,000 / 128 times at most where its workgroup has four waves of 32 keys at a time; each addition is off by 2^-24
    of the total at most.  Scores are products of few bits; their exponentials are off by 2^-18, generously."""
    m, dim, page, dtype = 100_000, 64, 32, DTYPE[suffix]
    q, k = torch.zeros(rows, 1, dim), torch.zeros(m, 1, dim)
    q[:, 0, 0], k[0, 0, 0] = 4.0, above / 4
    k[1:, 0, 0] = torch.randn(m - 1, generator=torch.Generator().manual_seed(3)) * 0.1
    q, k = q.to(dtype), k.to(dtype)
    scores = (q.double()[:, 0] @ k.double()[:, 0].t()).masked_fill(~torch.ones(rows, m, dtype=torch.bool).tril(m - rows), -math.inf)
    want = torch.logsumexp(scores, 1)
    out, lse = torch.empty_like(q, device="cuda"), torch.full((1, rows), 7.0, device="cuda")
    q, k = q.cuda(), k.cuda()
    q_offsets = oracle.offsets_of([rows]).cuda()
    if how == "packed":
        hip.attention_packed(suffix, q, k, k, q_offsets, oracle.offsets_of([m]).cuda(), out, lse, scale=1.0)
    else:
        table = torch.arange(m // page, dtype=torch.int32, device="cuda")[None]
        cache = k.view(m // page, page, 1, dim)
        hip.attention_paged(suffix, q, cache, cache, table, q_offsets, torch.tensor([m], dtype=torch.int32).cuda(), out, lse,
                            max_kv_length=m if how == "parts" else 1, scale=1.0)
    torch.cuda.synchronize()
    off = float((lse.cpu().double()[0] - want).abs().max())
    log(f"lse off by {off:.2e}")
    assert off <= (m / 128 + 16) * 2.0 ** -24 + 2.0 ** -18 + 4 * 2.0 ** -24 * above
