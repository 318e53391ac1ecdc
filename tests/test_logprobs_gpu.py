"""Log probabilities of given tokens: from logits and behind the product that keeps none, against their definition in 64 bits."""
import math

import numpy as np
import pytest
import torch

from helpers import make_model_folder

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -24  # half a float32 step, relative


@pytest.fixture(scope="module")
def ops():
    from abacus_b200.kernels import ops
    return ops


def plain(x, tokens, top):
    """(logprob, entropy, ids, values) of rows x (float64): the definition, row by row."""
    n, vocab = x.shape
    logprob, entropy = np.full(n, np.nan), np.full(n, np.nan)
    ids, values = np.full((n, top), -1, dtype=np.int64), np.full((n, top), np.nan)
    for r in range(n):
        row = x[r]
        if np.isnan(row).any() or (row == np.inf).any() or (row == -np.inf).all():
            continue
        m = row.max()
        logp = row - m - math.log(np.exp(row - m).sum())
        p = np.exp(logp)
        entropy[r] = -(p[p > 0] * logp[p > 0]).sum()
        if 0 <= tokens[r] < vocab:
            logprob[r] = logp[tokens[r]]
        ids[r] = np.lexsort((np.arange(vocab), -row))[:top]
        values[r] = logp[ids[r]]
    return logprob, entropy, ids, values


def compare(got, want, vocab):
    """Every term e^(x - m) is off by 2^-22 (the exponential) and |x - m| 2^-23 (its argument), where sum p |x - m| is at most
    log V; a thread adds up to V / 512 of them, then 13 joins: l is off by (V / 512 + 13 + 4 + 2 log V) half steps at most. The
    logarithm, two subtractions and the sum for the entropy add 3 half steps of the numbers they give."""
    logprob, entropy, ids, values = got
    w_logprob, w_entropy, w_ids, w_values = want
    of_l = HALF * (vocab / 512 + 17 + 2 * math.log(max(vocab, 2)) + math.log(max(vocab, 2)))

    def near(a, b, extra):
        assert np.array_equal(np.isnan(a), np.isnan(b)) and np.array_equal(a == -np.inf, b == -np.inf)
        ok = np.isfinite(b)
        assert (np.abs(a[ok] - b[ok]) <= of_l * extra + 4 * HALF * np.abs(b[ok]) + 1e-30).all(), np.abs(a[ok] - b[ok]).max()
    near(logprob, w_logprob, 1)
    if entropy is not None:
        near(entropy, w_entropy, 2 + math.log(max(vocab, 2)))
    if ids is not None:
        assert np.array_equal(ids, w_ids)
        near(values, w_values, 1)


def run(ops, x, tokens, top, entropy=True):
    n = x.shape[0]
    logprob = torch.full((n + 1,), 7.0, device="cuda")
    h = torch.full((n + 1,), 7.0, device="cuda") if entropy else None
    ids = torch.full((n + 1, top), 9, dtype=torch.int32, device="cuda") if top else None
    values = torch.full((n + 1, top), 7.0, device="cuda") if top else None
    ops.token_logprobs(x, torch.tensor(tokens, dtype=torch.int32, device="cuda"), logprob, entropy=h, top_ids=ids, top_logprobs=values, n_rows=n)
    assert float(logprob[n]) == 7.0 and (h is None or float(h[n]) == 7.0) and (not top or (int(ids[n, 0]) == 9 and float(values[n, 0]) == 7.0))
    return (logprob[:n].double().cpu().numpy(), h[:n].double().cpu().numpy() if entropy else None,
            ids[:n].cpu().numpy() if top else None, values[:n].double().cpu().numpy() if top else None)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n, vocab, top", [(1, 1, 1), (3, 2, 2), (2, 7, 0), (5, 33, 20), (1, 1000, 64), (4, 4099, 5), (2, 8195, 64), (3, 16391, 1),
                                           (40, 5003, 3), (7, 50261, 20), (2, 151936, 64), (700, 4097, 2), (1, 262147, 20)])
def test_logprobs_of_logits(ops, dtype, n, vocab, top):
    """Rows of every length class (one CTA, clusters of every size), odd vocabularies whose rows start anywhere, ties (bfloat16)."""
    g = torch.Generator(device="cuda").manual_seed(vocab + n)
    x = (torch.randn((n, vocab), generator=g, device="cuda") * 3.0).to(dtype)
    tokens = torch.randint(vocab, (n,), generator=g, device="cuda").tolist()
    compare(run(ops, x, tokens, top), plain(x.double().cpu().numpy(), tokens, top), vocab)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_that_are_masked_or_no_distribution(ops, dtype):
    """Masks of -inf (few tokens left, one, none), of the type's lowest value (everywhere too), NaN and infinities, constant rows,
    rising and falling ones (every element the largest so far), sharp ones; tokens outside the vocabulary."""
    vocab, low = 9001, torch.finfo(dtype).min
    x = torch.randn((16, vocab), generator=torch.Generator().manual_seed(1)) * 2.0
    x[1, torch.arange(vocab) % 1000 != 7] = -math.inf  # ten left, fewer than are asked for
    x[2] = -math.inf
    x[2, 8999] = 3.0
    x[3] = -math.inf
    x[4, 100:] = low
    x[5] = low
    x[6, 4000] = math.nan
    x[7, 17] = math.inf
    x[8] = 1.25
    x[9] = torch.arange(vocab) / 64.0
    x[10] = -torch.arange(vocab) / 64.0
    x[11, 123] = 60.0
    x[12, 5:] = -math.inf
    x[13] = 0.0
    x[13, 1::2] = -0.0
    x[14] = torch.where(torch.arange(vocab) % 3 == 0, 5.0, -5.0)
    x[15] = -1e30 if dtype == torch.float32 else -2.0 ** 90
    x = x.to(dtype).cuda()
    tokens = [5, 7, 8999, 3, 50, 6, 0, 17, 9000, 9000, 0, 123, 6, -1, vocab, 1 << 30]
    for top in (0, 1, 20, 64):
        compare(run(ops, x, tokens, top), plain(x.double().cpu().numpy(), tokens, top), vocab)
    # and the same rows as one of few, where a cluster takes each (another way through the kernel)
    for r in range(16):
        one = x[r:r + 1, :].repeat(1, 4)
        compare(run(ops, one, tokens[r:r + 1], 20), plain(one.double().cpu().numpy(), tokens[r:r + 1], 20), 4 * vocab)


def test_strides_streams_and_graphs(ops):
    """Rows of a wider matrix that start at every offset from a 16-byte boundary; on another stream; captured, twice, and replayed on
    new logits; the same call twice gives the same bits."""
    wide = torch.randn((6, 5 * 7001), generator=torch.Generator().manual_seed(3)).cuda()
    for at in range(5):
        x = wide[:, at:at + 7001]
        compare(run(ops, x, [1, 2, 3, 4, 5, 6], 4), plain(x.double().cpu().numpy(), [1, 2, 3, 4, 5, 6], 4), 7001)
    half = wide.to(torch.bfloat16)
    for at in range(9):
        x = half[:, at:at + 6003]
        compare(run(ops, x, [1, 2, 3, 4, 5, 6], 4), plain(x.double().cpu().numpy(), [1, 2, 3, 4, 5, 6], 4), 6003)
    x, tokens = wide[:, :30000].contiguous(), torch.arange(6, dtype=torch.int32, device="cuda")
    outs = [[torch.zeros(6, device="cuda"), torch.zeros(6, device="cuda"), torch.zeros((6, 8), dtype=torch.int32, device="cuda"), torch.zeros((6, 8), device="cuda")]
            for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.token_logprobs(x, tokens, *outs[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for out in outs:
        ops.token_logprobs(x, tokens, *out)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.token_logprobs(x, tokens, *out)
        graphs.append(g)
    x.mul_(0.5)
    for g in graphs * 2:
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    compare([t.double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy() for t in outs[0]],
            plain(x.double().cpu().numpy(), list(range(6)), 8), 30000)


def test_refusals(ops):
    x, t, out = torch.zeros((3, 50), device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(3, device="cuda")
    ids, values = torch.zeros((3, 65), dtype=torch.int32, device="cuda"), torch.zeros((3, 65), device="cuda")
    with pytest.raises(ops.KernelRefused):
        ops.token_logprobs(x, t, out, top_ids=ids, top_logprobs=values)  # more than 64
    with pytest.raises(ops.KernelRefused):
        ops.token_logprobs(x, t, out, top_ids=ids[:, :51].contiguous(), top_logprobs=values[:, :51].contiguous())  # more than there are
    with pytest.raises(AssertionError):
        ops.token_logprobs(x, t, out, top_ids=ids[:, :5].contiguous())
    with pytest.raises(AssertionError):
        ops.token_logprobs(x, t.long(), out)
    with pytest.raises(ops.KernelError):
        ops.token_logprobs(x.half(), t, out)
    with pytest.raises(ops.KernelError):
        ops.token_logprobs(x.cpu(), t, out)
    ops.token_logprobs(x, t, out, n_rows=0)
    from abacus_b200.parts import Workspace
    ws = Workspace(torch.device("cuda"))
    with pytest.raises(ops.KernelRefused):
        ops.gemm_tc_logprobs(torch.zeros((3, 12), dtype=torch.bfloat16, device="cuda"), torch.zeros((9, 12), dtype=torch.bfloat16, device="cuda"),
                             t, out, None, ws)
    ops.gemm_tc_logprobs(torch.zeros((3, 16), dtype=torch.bfloat16, device="cuda"), torch.zeros((9, 16), dtype=torch.bfloat16, device="cuda"),
                         t, out, None, ws, m=0)


@pytest.mark.parametrize("m, vocab, k", [(1, 1, 8), (1, 300, 64), (5, 257, 72), (37, 5003, 200), (128, 1024, 128), (129, 999, 64), (256, 4097, 264),
                                         (300, 20011, 1024), (2049, 3001, 136), (2500, 515, 192), (33, 2000, 2048), (70, 3333, 2056), (40, 1500, 4096),
                                         (16390, 260, 64), (1, 5000, 1024), (16, 20000, 1160), (17, 37777, 648), (33, 12001, 4096), (50, 30011, 2400),
                                         (64, 151936, 640), (64, 22003, 4160)])
def test_logprobs_behind_the_product(ops, m, vocab, k):
    """Row tiles that end anywhere, groups of them, vocabularies that end inside a tile, fewer tiles than pairs of SMs, K that is one
    segment, two, or ends inside a block; few rows against large matrices, which run on a kernel of their own; rows beyond m are left alone.

    A logit is off by K half steps of sum |x w| (the tensor cores cut off instead of rounding: a step of 2^-23 of the running sum for
    every 16 products, counted here as K / 16 + 16 of them); a log probability by twice that of the logits that matter."""
    from abacus_b200.parts import Workspace
    g = torch.Generator(device="cuda").manual_seed(m + vocab)
    x = torch.randn((m + 1, k), generator=g, device="cuda").to(torch.bfloat16)
    w = (torch.randn((vocab, k), generator=g, device="cuda") * (3.0 / math.sqrt(k))).to(torch.bfloat16)
    tokens = torch.randint(vocab, (m + 1,), generator=g, device="cuda", dtype=torch.int32)
    tokens[0], tokens[-1] = vocab - 1, -1
    if m > 2:
        tokens[1], tokens[2] = -1, vocab
    logprob, entropy = torch.full((m + 1,), 7.0, device="cuda"), torch.full((m + 1,), 7.0, device="cuda")
    ws = Workspace(torch.device("cuda"))
    for _ in range(2):
        ops.gemm_tc_logprobs(x, w, tokens, logprob, entropy, ws, m=m)
    assert float(logprob[m]) == 7.0 and float(entropy[m]) == 7.0
    logits = x[:m].double() @ w.double().t()
    scale = (x[:m].double().abs() @ w.double().abs().t()).amax(dim=1)
    logp = torch.log_softmax(logits, dim=1)
    h = -(logp.exp() * logp).sum(dim=1)
    off = scale * 2.0 ** -23 * (min(k, 2048) / 16 + 16) + HALF * (vocab / 2 + 40)
    valid = (tokens[:m] >= 0) & (tokens[:m] < vocab)
    given = logp.gather(1, tokens[:m].clamp(0, vocab - 1).long()[:, None])[:, 0]
    assert torch.equal(torch.isnan(logprob[:m]), ~valid)
    assert ((logprob[:m].double() - given).abs()[valid] <= 2 * off[valid] + 4 * HALF * given.abs()[valid]).all()
    assert ((entropy[:m].double() - h).abs() <= 2 * off * (2 + math.log(vocab + 1)) + 4 * HALF * h).all()
    again = torch.zeros(m, device="cuda")
    ops.gemm_tc_logprobs(x[:m], w, tokens[:m].contiguous(), again, None, ws)
    assert torch.equal(again.nan_to_num(3.0), logprob[:m].nan_to_num(3.0))


def test_logprobs_behind_the_product_of_slices_and_of_what_is_not_finite(ops):
    """Operands inside wider matrices; a row with a NaN or an infinity gives NaN and leaves the others alone."""
    from abacus_b200.parts import Workspace
    ws = Workspace(torch.device("cuda"))
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn((50, 320), generator=g, device="cuda").to(torch.bfloat16)[:, 64:192]
    w = torch.randn((700, 256), generator=g, device="cuda").to(torch.bfloat16)[:, 8:136]
    tokens = torch.arange(50, dtype=torch.int32, device="cuda")
    out, h = torch.zeros(50, device="cuda"), torch.zeros(50, device="cuda")
    ops.gemm_tc_logprobs(x, w, tokens, out, h, ws)
    logp = torch.log_softmax(x.double() @ w.double().t(), dim=1)
    assert (out.double() - logp[torch.arange(50), torch.arange(50)]).abs().max() < 1e-3
    y = x.clone()
    y[3, 5], y[40, 0] = math.nan, math.inf
    bad, hb = torch.zeros(50, device="cuda"), torch.zeros(50, device="cuda")
    ops.gemm_tc_logprobs(y, w, tokens, bad, hb, ws)
    fine = torch.ones(50, dtype=torch.bool)
    fine[3] = fine[40] = False
    assert torch.equal(bad[fine], out[fine]) and torch.equal(hb[fine], h[fine]) and bad[~fine].isnan().all() and hb[~fine].isnan().all()


@pytest.mark.parametrize("name, dtype", [("A", "bfloat16"), ("B", "bfloat16"), ("D", "bfloat16"), ("B", "float32")])
def test_scores_through_the_library(tmp_path, name, dtype):
    """LM.score against the logits that the engine gives for the same tokens, with and without alternatives, in unequal batches larger than
    the cache, single tokens, and generate(logprobs=..) against the score of what it generated."""
    import abacus_b200
    folder = make_model_folder(tmp_path, name)
    lm = abacus_b200.LM(folder, dtype=dtype, max_tokens=512)
    rng = np.random.default_rng(0)
    vocab = lm.model.spec.vocab
    texts = [rng.integers(0, vocab, n).tolist() for n in (1, 2, 65, 200, 130, 17, 300)]
    for top in (0, 3):
        scores = lm.score(texts, top=top)
        for text, s in zip(texts, scores):
            assert s.tokens == text and len(s.logprobs) == len(s.entropies) == len(text) - 1
            if len(text) == 1:
                continue
            slot = lm.engine.open()
            logits = lm.engine.step([(slot, text, list(range(len(text) - 1)))]).double().cpu()
            lm.engine.close(slot)
            logp = torch.log_softmax(logits, dim=1)
            want = logp[torch.arange(len(text) - 1), torch.tensor(text[1:])].numpy()
            # the same float32 logits up to the order of their sums, and in bfloat16 up to flipped roundings on the way (helpers.assert_logits)
            off = 1e-3 if dtype == "float32" else 0.02 * float(logits.abs().max()) * 2
            assert np.abs(np.array(s.logprobs) - want).max() <= off
            assert abs(s.total - sum(s.logprobs)) < 1e-9
            if top:
                assert [len(t) for t in s.top] == [3] * (len(text) - 1)
                assert all(a[1] >= b[1] for t in s.top for a, b in zip(t, t[1:]))
                assert np.abs(np.array([t[0][1] for t in s.top]) - logp.max(dim=1).values.numpy()).max() <= off
    assert lm.engine.cache.free_pages == lm.engine.cache.n_pages
    requests = lm.generate([texts[1], texts[2]], max_new_tokens=6, temperature=0.0, stop_tokens=[], return_requests=True, logprobs=2)
    for r in requests:
        assert len(r.logprobs) == len(r.output) == 6 and all(t[0][0] == token for t, token in zip(r.top, r.output))  # greedy: the likeliest
        assert all(abs(t[0][1] - p) < 1e-6 for t, p in zip(r.top, r.logprobs))
        s = lm.score([list(r.prompt) + r.output])[0]
        off = 1e-3 if dtype == "float32" else 0.3
        assert np.abs(np.array(s.logprobs[-6:]) - np.array(r.logprobs)).max() < off
    plain_run = lm.generate([texts[1], texts[2]], max_new_tokens=6, temperature=0.0, stop_tokens=[])
    assert plain_run == [r.output for r in requests]
