"""Log probabilities behind the product at logits of every size, and to the last digits."""
import math

import pytest
import torch

from test_logprobs_gpu import HALF, ops  # noqa: F401  (ops is a fixture)

pytestmark = pytest.mark.gpu


def product(ops, x, w, tokens):  # noqa: F811
    from abacus_b200.parts import Workspace
    out = [torch.full((x.shape[0],), 7.0, device="cuda") for _ in range(2)]
    ops.gemm_tc_logprobs(x, w, torch.tensor(tokens, dtype=torch.int32, device="cuda"), *out, Workspace(torch.device("cuda")))
    return [t.double().cpu() for t in out]


@pytest.mark.parametrize("m, vocab, k", [(3, 5, 64), (200, 37, 64), (2, 300, 2056), (3, 5003, 1024), (7, 20011, 512), (1, 151937, 64),
                                         (140, 5003, 2056)])
def test_logits_of_any_size_that_are_finite(ops, m, vocab, k):  # noqa: F811
    """Rows whose logits all lie far below -1e30, far above 1e30, or at both ends of float32, with vocabularies that end inside a piece, in the
    kernels for few and for many rows: a row's logits are x[0] w[:, 0], exactly. The largest are alike (h of them), the others at
    least 2^80 below, so the log probability is -log h or -inf and the entropy log h, to the roundings of a logarithm and of sums of
    up to `vocab` / 100 ones (exact below 2^24). One -inf, or a NaN, makes the row NaN."""
    h = max(1, vocab // 3)
    for first, high, low in ((2.0 ** 53, -2.0 ** 53, -2.0 ** 55), (2.0 ** 53, 2.0 ** 54, -1.0), (2.0 ** 53, 2.0 ** 54, 2.0 ** 53),
                             (2.0 ** 63, 2.0 ** 63, -2.0 ** 64), (2.0 ** 64, -2.0 ** 62, -2.0 ** 63), (-2.0 ** 53, 1.0, 2.0 ** 53)):
        x, w = torch.zeros((m, k)), torch.zeros((vocab, k))
        x[:, 0], w[:, 0] = first, low
        w[torch.arange(h) * 3 % vocab, 0] = high
        x, w = x.to(torch.bfloat16).cuda(), w.to(torch.bfloat16).cuda()
        tokens = [(0 if r % 2 else vocab - 1) for r in range(m)]
        exact = (x[:1].double() @ w.double().t())[0].cpu()
        logp = torch.log_softmax(exact, dim=0)
        logprob, entropy = product(ops, x, w, tokens)
        want = logp[torch.tensor(tokens)].float().double()
        assert torch.equal(torch.isinf(logprob), torch.isinf(want))
        near = torch.isfinite(want)
        assert ((logprob - want).abs()[near] <= 4 * HALF * (want.abs()[near] + math.log(vocab))).all(), (first, high, low)
        assert ((entropy - math.log(h)).abs() <= 4 * HALF * math.log(vocab)).all(), (first, high, low, entropy)
        for bad in (-math.inf, math.nan):
            spoilt = w.clone()
            spoilt[1, 0] = bad * math.copysign(1.0, first)
            assert all(t.isnan().all() for t in product(ops, x, spoilt, tokens))


@pytest.mark.parametrize("m, vocab, k", [(64, 151936, 640), (1, 151937, 64), (5, 257, 72), (33, 12001, 4096), (37, 20011, 1024), (300, 20011, 1024),
                                         (129, 151936, 64), (2049, 3001, 136), (2500, 99999, 64), (70, 3333, 2056), (16390, 260, 64)])
def test_no_token_is_missing_or_counted_twice(ops, m, vocab, k):  # noqa: F811
    """Rows of zeros: every token has the log probability -log V and the entropy is log V. All sums are whole numbers below 2^24, so only
    the logarithm (a step off, two halves) and a rounding are: a single token too few or too many of 151,936 is 6.6e-6, the bound 2.2e-6."""
    x, w = torch.zeros((m, k), dtype=torch.bfloat16, device="cuda"), torch.ones((vocab, k), dtype=torch.bfloat16, device="cuda")
    logprob, entropy = product(ops, x, w, [r * 7919 % vocab for r in range(m)])
    log = math.log(vocab)
    assert max((logprob + log).abs().max(), (entropy - log).abs().max()) <= 3 * HALF * log < math.log1p(1 / vocab)


@pytest.mark.parametrize("m, vocab, k", [(3, 1003, 8192), (200, 700, 8192), (2, 5003, 12160), (70, 300, 12160)])
def test_a_long_k_is_added_up_in_segments(ops, m, vocab, k):  # noqa: F811
    """One token's logit is a sum S of a first product of 32 and many small ones, the others' are zero: the log probability of another is -S
    (beside e^-S V, which is taken in too). The tensor cores cut off a step of 2^-23 of the running sum at most for every 16 products:
    in a first segment of 1,024 that is 64 such steps of S at most, in the others, whose sums are small, less than one together, and eight
    roundings more for adding up. In one segment of 8,192 or more the small products lose half a step of S for each 16 on average."""
    g = torch.Generator().manual_seed(k)
    x, w = torch.ones((m, k), dtype=torch.bfloat16), torch.zeros((vocab, k), dtype=torch.bfloat16)
    w[5] = (torch.rand(k, generator=g) * 8.0 / k).to(torch.bfloat16)
    w[5, 0] = 32.0
    s = float(w[5].double().sum())
    logprob, _ = product(ops, x.cuda(), w.cuda(), [vocab - 1 - r % 2 for r in range(m)])
    want = -s - math.log1p((vocab - 1) * math.exp(-s))
    assert ((logprob - want).abs() <= s * 2.0 ** -23 * (64 + 1 + 8)).all(), float((logprob - want).abs().max()) / s * 2.0 ** 23
