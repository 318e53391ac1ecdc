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
