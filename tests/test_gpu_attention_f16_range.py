"""f16's narrow exponents: weights and score gradients that are small or large against 1 keep their bits.

Every tensor is compared as a whole, or in blocks of rows.  With u = 2^-11, f16's unit roundoff: a value that f16 holds as a normal
number is rounded by a part of at most u, by 0.41 u in the root mean square (a uniform error of half an ulp either way, mantissas
spread over their logarithm).  dQ and dK carry that of dS, that of the output within rowsum(dO O), and that of the
result; dV that of P and of the result.  The result's own is taken from the 64-bit value, since it is larger where results are
subnormal; what remains is at most sqrt(2) 0.41 u = 0.58 u of the tensor's norm, and 32-bit sums are far below.  Allowed: u.
"""
import math

import pytest
import torch

import attention_oracle as oracle
from gpu_util import log

pytestmark = pytest.mark.gpu

U = 2.0 ** -11


def rows(tokens, heads, dim, seed, gain=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(tokens, heads, dim, generator=g) * gain).half()


def formulas(q, k, v, dout, lengths, scale, causal=True):
    """dq, dk and dv in 64 bits; sequences of as many keys as rows, or one that is not causal."""
    dq, dk, dv = (torch.zeros(x.shape, dtype=torch.float64) for x in (q, k, v))
    group, at = q.shape[1] // k.shape[1], 0
    for n in lengths:
        r, c = slice(at, at + n), slice(at, at + n) if causal else slice(None)
        at += n
        for h in range(q.shape[1]):
            qh, kh, vh, do = (x.double() for x in (q[r, h], k[c, h // group], v[c, h // group], dout[r, h]))
            scores = qh @ kh.t() * scale
            if causal:
                scores.masked_fill_(torch.ones(n, n, dtype=torch.bool).triu(1), -math.inf)
            p = torch.softmax(scores, 1)
            dv[c, h // group] += p.t() @ do
            ds = do @ vh.t()
            ds = p * (ds - (p * ds).sum(1, keepdim=True)) * scale
            dq[r, h] = ds @ kh
            dk[c, h // group] += ds.t() @ qh
    return {"dq": dq, "dk": dk, "dv": dv}


def run(hip, q, k, v, dout, lengths, causal=True):
    o, ko = oracle.offsets_of(lengths).cuda(), oracle.offsets_of(lengths if causal else [k.shape[0]]).cuda()
    q, k, v, dout = (x.cuda() for x in (q, k, v, dout))
    out, lse = torch.empty_like(q), torch.empty(q.shape[1], q.shape[0], device="cuda")
    hip.attention_packed("f16", q, k, v, o, ko, out, lse, causal=causal)
    got = {"dq": torch.full_like(q, 7.0), "dk": torch.full_like(k, 7.0), "dv": torch.full_like(v, 7.0)}
    hip.attention_packed_backward("f16", q, k, v, out, lse, dout, o, ko, got["dq"], got["dk"], got["dv"], causal=causal)
    torch.cuda.synchronize()
    return got


def near(name, got, want):
    got = got.cpu().double()
    assert torch.isfinite(got).all(), f"{name}: not finite"
    size = float(want.norm())
    off, own = float((got - want).norm()) / size, float((want.half().double() - want).norm()) / size
    log(f"{name}: off by {off:.2e} of its size, rounding alone {own:.2e}, allowed {own + U:.2e}")
    assert off <= own + U, name


@pytest.mark.parametrize("width", [1.0, 1e-2, 1e-3, 1e-4])
@pytest.mark.parametrize("lengths,heads,kv_heads,dim", [([3000], 2, 1, 128), ([1700, 1300], 4, 4, 64), ([2600], 3, 1, 80)])
def test_gradients_of_small_output_gradients(hip, dev, lengths, heads, kv_heads, dim, width):
    """Rows over thousands of keys, dO of any width that f16 holds."""
    n = sum(lengths)
    q, k, v, dout = rows(n, heads, dim, 1), rows(n, kv_heads, dim, 2), rows(n, kv_heads, dim, 3), rows(n, heads, dim, 4, width)
    want = formulas(q, k, v, dout, lengths, dim ** -0.5)
    got = run(hip, q, k, v, dout, lengths)
    for name in want:
        near(name, got[name], want[name])


def test_gradients_of_small_values(hip, dev):
    """dP is small where the values are."""
    n, dim = 2500, 64
    q, k, v, dout = rows(n, 2, dim, 1), rows(n, 1, dim, 2), rows(n, 1, dim, 3, 1e-2), rows(n, 2, dim, 4, 1e-2)
    want = formulas(q, k, v, dout, [n], dim ** -0.5)
    got = run(hip, q, k, v, dout, [n])
    for name in want:
        near(name, got[name], want[name])


@pytest.mark.parametrize("heads,kv_heads", [(2, 1), (3, 3)])
def test_gradients_of_large_output_gradients(hip, dev, heads, kv_heads):
    """dS past 65,504, the largest f16, where dQ and dK are not: a scaled loss, large values and small keys and rows."""
    n, m, dim = 300, 8, 128
    q, k, v, dout = rows(n, heads, dim, 1, 0.02), rows(m, kv_heads, dim, 2, 0.02), rows(m, kv_heads, dim, 3, 8.0), rows(n, heads, dim, 4, 4000.0)
    want = formulas(q, k, v, dout, [n], dim ** -0.5, causal=False)
    assert all(float(x.abs().max()) < 65504 for x in (want["dq"], want["dk"]))
    got = run(hip, q, k, v, dout, [n], causal=False)
    for name in ("dq", "dk"):
        near(name, got[name], want[name])


@pytest.mark.parametrize("rising", [True, False])
@pytest.mark.parametrize("lengths,heads,kv_heads", [([2000], 2, 1), ([900, 1100], 3, 3)])
def test_gradients_of_rows_of_all_sizes(hip, dev, lengths, heads, kv_heads, rising):
    """dO from 2^-13 to 2^7 along the rows: what a few rows' sums are scaled to does not stay right for the next."""
    n, dim = sum(lengths), 64
    q, k, v, dout = rows(n, heads, dim, 1), rows(n, kv_heads, dim, 2), rows(n, kv_heads, dim, 3), rows(n, heads, dim, 4)
    exponent = torch.linspace(-13.0, 7.0, n).floor()
    dout = (dout.float() * torch.exp2(exponent if rising else exponent.flip(0))[:, None, None]).half()
    want = formulas(q, k, v, dout, lengths, dim ** -0.5)
    got = run(hip, q, k, v, dout, lengths)
    for at in range(0, n, 250):
        near(f"dq {at}", got["dq"][at:at + 250], want["dq"][at:at + 250])
    for name in ("dk", "dv"):
        near(name, got[name], want[name])


# ---- weights far below a row's largest -------------------------------------------------------------
def one_key_above(m, dim, n, seed=5):
    """n rows whose score with key 0 is 17 above those with the other m - 1, whose weights together are m e^-17."""
    q, k = torch.zeros(n, 1, dim), torch.zeros(m, 1, dim)
    q[:, 0, 0], k[0, 0, 0] = 4.0, 4.25
    k[1:, 0, 0] = torch.randn(m - 1, generator=torch.Generator().manual_seed(seed)) * 0.1
    v = 1.0 + rows(m, 1, dim, seed + 1, 0.1).float()
    v[0] = 0.0
    return q.half(), k.half(), v.half()


def check_one_key_above(q, k, v, new, out, lse):
    """Weights are off by a part of u, or by what the range leaves: 2^-25 of a weight that is at least 2^7 where the row's largest
    is 1, 2^-32 of the row's sum each.  (32-bit exponentials and sums as in the other tests: 2^-17.)"""
    m = k.shape[0]
    scores = q.double()[:, 0] @ k.double()[:, 0].t()
    scores = scores.masked_fill(~torch.ones(new, m, dtype=torch.bool).tril(m - new), -math.inf)
    weights, values = torch.softmax(scores, 1), v.double()[:, 0]
    want = weights @ values
    bound = (2 * U + 2.0 ** -17) * want + 2.0 ** -32 * values.abs().sum(0) + 2.0 ** -25
    off = (out.cpu().double()[:, 0] - want).abs()
    log(f"off by {float((off / want).max()):.2e} of the output, allowed {float((bound / want).min()):.2e}")
    assert (off <= bound).all()
    assert (lse.cpu().double()[0] - torch.logsumexp(scores, 1)).abs().max() <= 2.0 ** -15


@pytest.mark.parametrize("n", [1, 130])
def test_packed_weights_far_below_the_largest(hip, dev, n):
    m, dim = 100_000, 64
    q, k, v = one_key_above(m, dim, n)
    out, lse = torch.full((n, 1, dim), 7.0, dtype=torch.float16, device="cuda"), torch.full((1, n), 7.0, device="cuda")
    hip.attention_packed("f16", q.cuda(), k.cuda(), v.cuda(), oracle.offsets_of([n]).cuda(), oracle.offsets_of([m]).cuda(), out, lse,
                         scale=1.0)
    torch.cuda.synchronize()
    check_one_key_above(q, k, v, n, out, lse)


@pytest.mark.parametrize("n", [1, 60])
@pytest.mark.parametrize("parts", [False, True])
def test_paged_weights_far_below_the_largest(hip, dev, n, parts):
    """Rows of a narrow and a wide tile, in one part and in many."""
    m, dim, page = 100_000, 128, 32
    q, k, v = one_key_above(m, dim, n)
    pages = -(-m // page)
    caches = [torch.zeros(pages * page, 1, dim, dtype=torch.float16, device="cuda") for _ in range(2)]
    for cache, x in zip(caches, (k, v)):
        cache[:m] = x.cuda()
    caches = [c.view(pages, page, 1, dim) for c in caches]
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    out, lse = torch.full((n, 1, dim), 7.0, dtype=torch.float16, device="cuda"), torch.full((1, n), 7.0, device="cuda")
    hip.attention_paged("f16", q.cuda(), *caches, table, oracle.offsets_of([n]).cuda(), torch.tensor([m], dtype=torch.int32).cuda(), out,
                        lse, max_kv_length=m if parts else 1, scale=1.0)
    torch.cuda.synchronize()
    check_one_key_above(q, k, v, n, out, lse)
