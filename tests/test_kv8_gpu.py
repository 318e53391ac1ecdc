"""Keys and values in 8 bits: what the cache holds, to the bit; attention to it against 64 bits; models through the engine with it."""
import math

import numpy as np
import pytest
import torch

from helpers import make_model_folder

pytestmark = pytest.mark.gpu
TOP = {"int8": 127.0, "e4m3": 448.0}


@pytest.fixture(scope="module")
def ops():
    from abacus_b200.kernels import ops
    return ops


def held(x, form):
    """What a cache holds of a sequence's keys or values x [tokens, heads, dim] (bfloat16 numbers as float64): whole blocks of 16 as float32(q)
    times the float32 scale, the rest as it came. float32 numbers."""
    out = x.to(torch.float32).clone()
    for lo in range(0, len(x) // 16 * 16, 16):
        block = x[lo:lo + 16]
        most = block.abs().amax(dim=(0, 2))
        q = block * TOP[form] / torch.where(most > 0, most, torch.ones_like(most))[None, :, None]  # exact where it is a tie: 64 bits
        q = q.round() if form == "int8" else q.to(torch.float32).to(torch.float8_e4m3fn).to(torch.float64)
        scale = most.to(torch.float32) / TOP[form]
        block = q.to(torch.float32) * scale[None, :, None]
        block[:, ~torch.isfinite(most)] = math.nan
        out[lo:lo + 16] = block
    return out


class Run:
    """An 8-bit cache of one layer, sequences that grow in it, and all that they have brought (float64, on the host). What the cache
    must not read is filled with NaN patterns first."""

    def __init__(self, heads, kv_heads, dim, form, slots=6, pages=40, window=None, max_context=1 << 14):
        from abacus_b200.cache import CacheNeed, SequenceCache
        from abacus_b200.parts import Workspace
        self.heads, self.kv_heads, self.dim, self.form, self.window = heads, kv_heads, dim, form, window
        self.cache = SequenceCache([CacheNeed(kv_heads, dim, window)], [None], pages * 64, torch.bfloat16, "cuda", max_slots=slots,
                                   max_context=max_context, form=form)
        self.kv = self.cache.views[0].kv
        self.kv.open.fill_(math.nan)
        self.kv.scales.fill_(math.nan)
        self.kv.k.view(torch.uint8).fill_(0x7f), self.kv.v.view(torch.uint8).fill_(0xff)
        self.ws = Workspace(torch.device("cuda"))
        self.brought = {}
        self.g = torch.Generator().manual_seed(heads * 1000 + dim)

    def open(self):
        slot = self.cache.open_slot()
        self.brought[slot] = [torch.zeros((0, self.kv_heads, self.dim), dtype=torch.float64) for _ in range(2)]
        return slot

    def rows(self, n, spread=1.0):
        x = torch.randn((n, (self.heads + 2 * self.kv_heads) * self.dim), generator=self.g) * spread
        return x.to(torch.bfloat16)

    def batch(self, news):
        """[(slot, tokens)] -> a filled step; room is made and the lengths go on."""
        from abacus_b200.engine.batch import Sequence, StepBatch
        seqs = []
        for slot, n in news:
            start = self.cache.length[slot]
            self.cache.reserve(slot, start + n)
            self.cache.advance(slot, n)
            seqs.append(Sequence(slot, [0] * n, start, []))
        return StepBatch(sum(n for _, n in news), len(news), 1, "cuda").fill(seqs, exact=True)

    def write(self, ops, news, qkv):
        batch, at = self.batch(news), 0
        ops.kv8_write(qkv.cuda(), self.heads, self.kv_heads, self.dim, batch, self.kv)
        for slot, n in news:
            for j in range(2):
                lo = (self.heads + j * self.kv_heads) * self.dim
                x = qkv[at:at + n, lo:lo + self.kv_heads * self.dim].to(torch.float64).view(n, self.kv_heads, self.dim)
                self.brought[slot][j] = torch.cat([self.brought[slot][j], x])
            at += n
        return batch

    def read(self, ops, batch, dtype=torch.float32):
        counts = [-(-(s.start + len(s.tokens)) // 64) for s in batch.sequences]
        first = np.concatenate([[1], 1 + np.cumsum(counts)])
        k, v = (torch.full((int(first[-1]) + 2, self.kv_heads, 64, self.dim), 7.0, dtype=dtype, device="cuda") for _ in range(2))
        ops.kv8_read(self.kv, batch, torch.tensor(first, dtype=torch.int32, device="cuda"), k, v)
        k, v = k.cpu(), v.cpu()
        for t in (k, v):  # pages before and behind the sequences' own are left alone
            assert (t[0] == 7.0).all() and (t[int(first[-1]):] == 7.0).all()
        got = []
        for i, s in enumerate(batch.sequences):
            n = s.start + len(s.tokens)
            pair = [t[first[i]:first[i + 1]].permute(0, 2, 1, 3).reshape(-1, self.kv_heads, self.dim) for t in (k, v)]
            assert all((t[n:] == 0).all() for t in pair)
            got.append([t[:n] for t in pair])
        return got

    def check(self, ops, batch):
        for dtype in (torch.float32, torch.bfloat16):
            for s, pair in zip(batch.sequences, self.read(ops, batch, dtype)):
                for got, x in zip(pair, self.brought[s.slot]):
                    want = held(x, self.form).to(dtype)
                    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.5), want.nan_to_num(0.5))

    def attend(self, ops, batch, qkv):
        """Against 64 bits. The output is rounded to bfloat16 (2^-8 at most), the weights to float16 (2^-11 at most, of sum p |v|; what is
        2^-14 below the largest contribution to within 2^-25 of that, a key each); scores are float32 sums of exact products of q, whose
        elements are exact to 2^-25 of the largest, so that weights are off by 2^-14 beside."""
        n = batch.n_rows
        scale = self.dim ** -0.5
        out = torch.full((n + 1, self.heads * self.dim), 7.0, dtype=torch.bfloat16, device="cuda")
        ops.attention_kv8(qkv.cuda(), out, self.heads, self.kv_heads, self.dim, scale, self.window, batch, self.kv, self.ws)
        assert (out[n] == 7.0).all()
        again = torch.zeros_like(out)
        ops.attention_kv8(qkv.cuda(), again, self.heads, self.kv_heads, self.dim, scale, self.window, batch, self.kv, self.ws)
        assert torch.equal(out[:n], again[:n])
        at = 0
        for s in batch.sequences:
            keys, values = (held(x, self.form).to(torch.float64) for x in self.brought[s.slot])
            for t in range(len(s.tokens)):
                pos = s.start + t
                lo = max(0, pos - self.window + 1) if self.window else 0
                q = qkv[at, :self.heads * self.dim].to(torch.float64).view(self.kv_heads, -1, self.dim)
                k, v = keys[lo:pos + 1].transpose(0, 1), values[lo:pos + 1].transpose(0, 1)
                p = torch.softmax(q @ k.transpose(1, 2) * scale, dim=-1)
                want, size = p @ v, p @ v.abs()
                largest = (p[..., None] * v.abs()[:, None]).amax(dim=(2, 3))[..., None]
                tol = 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -13) * size + (pos + 1 - lo) * 2.0 ** -24 * largest
                got = out[at].double().cpu().view(self.kv_heads, -1, self.dim)
                assert torch.isfinite(got).all() and ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max()
                at += 1


SHAPES = [(1, 1, 64), (4, 2, 128), (8, 1, 64), (14, 2, 64), (9, 1, 128), (32, 2, 128), (20, 1, 64), (24, 8, 128), (33, 1, 128)]


@pytest.mark.parametrize("form", ["int8", "e4m3"])
@pytest.mark.parametrize("heads, kv_heads, dim", SHAPES)
def test_cache_and_attention_over_many_steps(ops, heads, kv_heads, dim, form):
    """Prompts of every kind of length, portions that begin and end anywhere in a block, single tokens through whole blocks, slots used
    again over what other sequences left, several sequences a step: what the cache holds is what the definition says, to the bit, and
    attention to it is right."""
    run = Run(heads, kv_heads, dim, form)
    a, b, c, d = (run.open() for _ in range(4))
    steps = [[(a, 1), (b, 16), (c, 70), (d, 15)], [(a, 14), (b, 1), (c, 40), (d, 1)], [(a, 1), (b, 1), (c, 1), (d, 1)], [(c, 17), (a, 2)],
             [(d, 3), (b, 130)], [(a, 33), (b, 4), (c, 1), (d, 64)], [(b, 5)]]
    for i, news in enumerate(steps):
        qkv = run.rows(sum(n for _, n in news), spread=1.0 + i)
        batch = run.write(ops, news, qkv)
        run.check(ops, batch)
        run.attend(ops, batch, qkv)
    run.cache.close_slot(b)
    run.brought.pop(b)
    b = run.open()
    for i in range(20):
        news = [(b, 1), (a, 1), (c, 1)][:1 + i % 3]
        qkv = run.rows(len(news))
        batch = run.write(ops, news, qkv)
        assert batch.is_decode
        if i % 4 == 3:
            run.check(ops, batch)
            run.attend(ops, batch, qkv)


@pytest.mark.parametrize("form", ["int8", "e4m3"])
@pytest.mark.parametrize("lengths, new", [([3000], 1), ([5000, 1, 17, 640], 1), ([129] * 40, 1), ([700, 64, 63, 65], 7), ([2, 1500], 1),
                                          ([40] * 600, 1)])
def test_attention_over_long_and_unequal_contexts(ops, lengths, new, form):
    """Pairs shared by many CTAs, CTAs with many pairs, more rows than a launch takes."""
    run = Run(8, 2, 64, form, slots=len(lengths), pages=sum(-(-(n + new) // 64) for n in lengths) + 2)
    slots = [run.open() for _ in lengths]
    for at in range(0, len(slots), 100):
        news = list(zip(slots, lengths))[at:at + 100]
        run.write(ops, news, run.rows(sum(n for _, n in news)))
    news = [(s, new) for s in slots]
    qkv = run.rows(new * len(slots), spread=2.0)
    batch = run.write(ops, news, qkv)
    if len(lengths) < 100:
        run.check(ops, batch)
    run.attend(ops, batch, qkv)


@pytest.mark.parametrize("window", [1, 15, 16, 64, 100, 200])
def test_attention_under_a_window_with_a_ring_of_pages(ops, window):
    """A windowed group keeps a ring of pages: prompts longer than the ring, then single tokens round it several times."""
    run = Run(6, 2, 64, "int8", slots=3, pages=20, window=window, max_context=1024)
    assert run.kv.ring_pages
    a, b = run.open(), run.open()
    run.write(ops, [(a, 500), (b, 3)], run.rows(503))
    for i in range(150):
        qkv = run.rows(2)
        batch = run.write(ops, [(a, 1), (b, 1)], qkv)
        if i % 7 == 0:
            run.attend(ops, batch, qkv)
    out = torch.zeros((2, 6 * 64), dtype=torch.bfloat16, device="cuda")
    for too_wide in (None, run.kv.ring_pages * 64 + 1):
        with pytest.raises(ops.KernelRefused, match="ring"):
            ops.attention_kv8(qkv.cuda(), out, 6, 2, 64, 0.125, too_wide, batch, run.kv, run.ws)
    with pytest.raises(ops.KernelRefused):
        ops.kv8_read(run.kv, batch, torch.zeros(3, dtype=torch.int32, device="cuda"), *(torch.zeros((1, 2, 64, 64), device="cuda") for _ in range(2)))


@pytest.mark.parametrize("form", ["int8", "e4m3"])
def test_numbers_of_every_size(ops, form):
    """Blocks of zeros, of halves (ties between steps), of the smallest and the largest numbers, with one number that dwarfs the others, and
    with one that is not finite (which reads back as NaN, its block alone)."""
    run = Run(2, 1, 64, form, slots=2, pages=8)
    a = run.open()
    qkv = run.rows(16 * 12)
    x = qkv[:, 2 * 64:].view(12, 16, 2, 64)
    x[0] = 0.0
    x[1] = torch.randint(-4, 5, (16, 2, 64), generator=run.g).to(torch.bfloat16) * 0.5
    x[2] = torch.randint(-255, 256, (16, 2, 64), generator=run.g).to(torch.bfloat16)
    x[3] *= 1e-39
    x[4] *= 1e-30
    x[5] *= 1e30
    x[6, 3, :, 5] = 3e38
    x[7, 2, 0, 7] = math.inf
    x[8, 0, 1, 0] = math.nan
    x[9] *= 2.0 ** -120
    x[10] = torch.where(torch.arange(64) % 2 == 0, 126.0, 252.0).to(torch.bfloat16)
    batch = run.write(ops, [(a, 16 * 12)], qkv)
    for got, want in zip(run.read(ops, batch)[0], run.brought[a]):
        want = held(want, form)
        assert torch.equal(got.isnan(), want.isnan())
        blocks, wanted = got.view(12, -1).nan_to_num(0.5), want.view(12, -1).nan_to_num(0.5)
        for i in range(12):
            if i == 3:  # below 2^-126 the scale itself has few digits: the numbers are right to a scale's last digit
                assert (blocks[i] - wanted[i]).abs().max() <= 128 * 2.0 ** -149 + wanted[i].abs().max() * 2.0 ** -7
            else:
                assert torch.equal(blocks[i], wanted[i]), i


@pytest.mark.parametrize("form", ["int8", "e4m3"])
@pytest.mark.parametrize("heads, kv_heads, dim, norms, angles", [(4, 2, 128, True, True), (5, 1, 64, True, False), (7, 7, 64, False, True), (2, 1, 128, False, False)])
def test_a_decode_step_prepared_on_its_way(ops, heads, kv_heads, dim, norms, angles, form):
    """kv8_write(prepare=..) leaves the bits that qkv_prep and kv8_write leave, through whole blocks, padded rows alone; several tokens a
    sequence and positions beyond the table are refused."""
    from abacus_b200.engine.batch import Sequence, StepBatch
    runs = [Run(heads, kv_heads, dim, form, slots=3, pages=12) for _ in range(2)]
    g = torch.Generator(device="cuda").manual_seed(dim + heads)
    q_norm, k_norm = (1.0 + 0.2 * torch.randn(dim, generator=g, device="cuda") for _ in range(2)) if norms else (None, None)
    cos = sin = None
    if angles:
        a = torch.rand((256, dim // 2), generator=g, device="cuda") * 6.0
        cos, sin = a.cos(), a.sin()
    prepare = dict(q_norm=q_norm, k_norm=k_norm, eps=1e-6, cos=cos, sin=sin)
    assert ops.kv8_write_prepares(torch.zeros(8, dtype=torch.bfloat16, device="cuda"), cos, sin, q_norm, k_norm, dim, False, dim)
    width = (heads + 2 * kv_heads) * dim
    starts = (0, 9, 15)
    for run in runs:
        for s in starts:
            slot = run.open()
            if s:
                run.g.manual_seed(s)
                run.write(ops, [(slot, s)], run.rows(s))
    for i in range(40):
        qkv = torch.randn((4, width), generator=g, device="cuda").to(torch.bfloat16)
        rows = []
        for run, fused in zip(runs, (True, False)):
            batch = StepBatch(4, 4, 1, "cuda").fill([Sequence(j, [0], s + i, []) for j, s in enumerate(starts)])
            for j, s in enumerate(starts):
                run.cache.reserve(j, s + i + 1)
            x = qkv.clone()
            if fused:
                ops.kv8_write(x, heads, kv_heads, dim, batch, run.kv, prepare=prepare)
            else:
                ops.qkv_prep(x, heads, kv_heads, dim, batch, q_norm, k_norm, 1e-6, cos, sin, dim if angles else 0, False, None)
                ops.kv8_write(x, heads, kv_heads, dim, batch, run.kv)
            rows.append(x)
        assert torch.equal(rows[0][:3, :heads * dim], rows[1][:3, :heads * dim]) and torch.equal(rows[0][3], qkv[3])
        bits = [(r.kv.k.view(torch.uint8), r.kv.v.view(torch.uint8), r.kv.scales.view(torch.int32)) for r in runs]
        assert all(torch.equal(x, y) for x, y in zip(*bits))
        for j, s in enumerate(starts):  # the open block's tokens (behind its end anything may lie)
            n = (s + i + 1) % 16
            assert torch.equal(runs[0].kv.open[j, :, :, :n].view(torch.int16), runs[1].kv.open[j, :, :, :n].view(torch.int16))
    with pytest.raises(ops.KernelRefused, match="single tokens"):
        several = StepBatch(2, 1, 1, "cuda").fill([Sequence(0, [0, 0], 40, [])], exact=True)
        ops.kv8_write(qkv, heads, kv_heads, dim, several, runs[0].kv, prepare=prepare)
    if angles:
        with pytest.raises(ops.KernelError, match="rotary table"):
            far = StepBatch(1, 1, 1, "cuda").fill([Sequence(0, [0], 256, [])], exact=True)
            ops.kv8_write(qkv, heads, kv_heads, dim, far, runs[0].kv, prepare=prepare)


def test_padding_streams_and_graphs(ops):
    """A captured decode step of more rows than it brings: padded rows become zeros and write nothing; replayed for a step that closes
    blocks, with a second graph captured between; the attention call on another stream."""
    from abacus_b200.engine.batch import Sequence, StepBatch
    run = Run(4, 2, 128, "int8", slots=5, pages=30)
    slots = [run.open() for _ in range(3)]
    run.write(ops, [(s, n) for s, n in zip(slots, (30, 100, 14))], run.rows(144))
    batch = StepBatch(8, 8, 1, "cuda")
    batch.position_bound = 1024
    qkv = torch.zeros((8, 8 * 128), dtype=torch.bfloat16, device="cuda")
    out = torch.full((8, 4 * 128), 7.0, dtype=torch.bfloat16, device="cuda")

    def fill():
        batch.fill([Sequence(s, [0], run.cache.length[s], []) for s in slots])

    def call():
        ops.kv8_write(qkv, 4, 2, 128, batch, run.kv)
        ops.attention_kv8(qkv, out, 4, 2, 128, 128 ** -0.5, None, batch, run.kv, run.ws)
    graphs = []
    for i in range(6):
        for s in slots:
            run.cache.reserve(s, run.cache.length[s] + 1)
        rows = run.rows(3)
        qkv.fill_(math.nan)
        qkv[:3] = rows.cuda()
        fill()
        if i in (0, 3):
            call()  # a step run twice is the same step
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                call()
            graphs.append(g)
            out.fill_(7.0)
        graphs[i % len(graphs)].replay()
        assert (out[3:] == 0).all()
        got = out[:3].clone()
        for j, s in enumerate(slots):
            run.cache.advance(s, 1)
            for side in range(2):
                lo = (4 + 2 * side) * 128
                run.brought[s][side] = torch.cat([run.brought[s][side], rows[j, lo:lo + 256].to(torch.float64).view(1, 2, 128)])
        plain_batch = StepBatch(3, 3, 1, "cuda").fill([Sequence(s, [0], run.cache.length[s] - 1, []) for s in slots], exact=True)
        run.check(ops, plain_batch)
        run.attend(ops, plain_batch, rows)
        other = torch.zeros_like(out)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            ops.attention_kv8(qkv, other, 4, 2, 128, 128 ** -0.5, None, batch, run.kv, run.ws)
        torch.cuda.current_stream().wait_stream(stream)
        assert torch.equal(other[:3], got)
    assert not any(ops.kernel_status(out.device).tolist())


def test_a_page_or_slot_that_is_not_there_is_reported_and_touches_nothing(ops):
    """A page number outside the pool and a slot outside the cache: the status says so, and all accesses stay inside (page or slot 0)."""
    from abacus_b200.engine.batch import Sequence, StepBatch
    run = Run(2, 1, 64, "int8", slots=2, pages=4)
    a = run.open()
    qkv = run.rows(70)
    batch = run.write(ops, [(a, 70)], qkv)
    table = run.kv.page_table.clone()
    status = ops.kernel_status(torch.device("cuda", torch.cuda.current_device()))
    out = torch.zeros((70, 128), dtype=torch.bfloat16, device="cuda")
    for bad in (1 << 20, -1):
        run.kv.page_table[a, 0] = bad
        ops.attention_kv8(qkv.cuda(), out, 2, 1, 64, 0.125, None, batch, run.kv, run.ws)
        ops.kv8_write(qkv.cuda(), 2, 1, 64, batch, run.kv)
        assert status.tolist()[2] == 2
        status.zero_()
        run.kv.page_table.copy_(table)
    wrong = StepBatch(1, 1, 1, "cuda").fill([Sequence(9, [0], 5, [])], exact=True)
    before = [t.clone() for t in (run.kv.k, run.kv.scales.view(torch.int32), run.kv.open.view(torch.int16))]
    ops.kv8_write(qkv[:1].cuda(), 2, 1, 64, wrong, run.kv)
    assert status.tolist()[2] == 4 and all(torch.equal(x, y) for x, y in zip(before, (run.kv.k, run.kv.scales.view(torch.int32), run.kv.open.view(torch.int16))))
    status.zero_()


def test_refusals(ops):
    run = Run(4, 2, 64, "int8", slots=2, pages=4)
    a = run.open()
    qkv = run.rows(10)
    batch = run.write(ops, [(a, 10)], qkv)
    out = torch.zeros((10, 256), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ops.KernelRefused):
        ops.kv8_write(torch.zeros((10, 12 * 64), dtype=torch.bfloat16, device="cuda"), 4, 4, 64, batch, run.kv)  # not the cache's heads
    with pytest.raises(AssertionError):
        ops.kv8_write(qkv.float().cuda(), 4, 2, 64, batch, run.kv)
    with pytest.raises(AssertionError):
        ops.attention_kv8(qkv.cuda(), out[:5], 4, 2, 64, 0.1, None, batch, run.kv, run.ws)
    with pytest.raises(ops.KernelError):
        ops.kv8_write(qkv, 4, 2, 64, batch, run.kv)  # not on the GPU
    batch.max_len_after = 64 * 4 + 1
    with pytest.raises(ops.KernelRefused):
        ops.attention_kv8(qkv.cuda(), out, 4, 2, 64, 0.1, None, batch, run.kv, run.ws)


@pytest.mark.parametrize("form", ["int8", "e4m3"])
def test_models_through_the_engine(tmp_path, ops, form):
    """A model of heads of 128 with its cache in 8 bits: every layer's cache holds what its projections made, to the bit, and attention is
    right against 64 bits at every kind of step (whole prompts attend to their own keys as they came); captured steps give what plain launches
    give, portions of a prompt what single tokens give, to bfloat16's roundings; generation and scoring run; fewer bytes."""
    import abacus_b200
    folder = make_model_folder(tmp_path, "D")
    lm = abacus_b200.LM(folder, max_tokens=64 * 40, cache=form)
    plain_lm = abacus_b200.LM(folder, max_tokens=64 * 40)
    engine = lm.engine
    per_token = lambda e: sum(t.numel() * t.element_size() for g in e.cache.groups for t in (g.k, g.v, g.scales) if t is not None) / (64 * 40)
    assert per_token(engine) < 0.51 * per_token(plain_lm.engine)
    spec = lm.model.blocks[-1].mixer.spec
    rng = np.random.default_rng(1)
    a, b = engine.open(), engine.open()
    first, second = rng.integers(0, 515, 203).tolist(), rng.integers(0, 515, 90).tolist()
    logits = engine.step([(a, first[:150], [149]), (b, second[:5], [4])])
    ref = plain_lm.engine
    ra, rb = ref.open(), ref.open()
    want = ref.step([(ra, first[:150], [149]), (rb, second[:5], [4])])
    # a whole prompt attends to its keys as they came: the same model but for the attention kernel's order of sums
    assert (logits - want).abs().max() <= 0.02 * want.abs().max()
    engine.step([(a, first[150:200], [49]), (b, second[5:80], [74])])  # portions: the pages are read back
    engine.step([(a, first[200:203], [2]), (b, second[80:81], [0])])   # a few tokens: row by row
    n = engine.last_batch.n_rows
    qkv = lm.model.ws.get("qkv", (n, lm.model.blocks[-1].mixer.row), torch.bfloat16)[:n].clone()
    att = lm.model.ws.get("att", (n, spec.n_heads * 128), torch.bfloat16)[:n].clone()
    kv = engine.cache.views[-1].kv
    counts = [-(-engine.length(s) // 64) for s in (a, b)]
    firsts = torch.tensor([0, counts[0], sum(counts)], dtype=torch.int32, device="cuda")
    k, v = (torch.zeros((sum(counts), spec.n_kv_heads, 64, 128), device="cuda") for _ in range(2))
    ops.kv8_read(kv, engine.last_batch, firsts, k, v)
    row = 0
    for i, s in enumerate(engine.last_batch.sequences):
        keys, values = (t[firsts[i]:firsts[i + 1]].permute(1, 0, 2, 3).reshape(spec.n_kv_heads, -1, 128).double() for t in (k, v))
        for t in range(len(s.tokens)):
            q = qkv[row, :spec.n_heads * 128].double().view(spec.n_kv_heads, -1, 128)
            seen = s.start + t + 1
            p = torch.softmax(q @ keys[:, :seen].transpose(1, 2) * spec.scale, dim=-1)
            exact = p @ values[:, :seen]
            got = att[row].double().view_as(exact)
            assert ((got - exact).abs() <= 2.0 ** -8 * exact.abs() + 2.0 ** -10 * (p @ values[:, :seen].abs())).all()
            row += 1
    # decoded together: graphs against plain launches
    bare = abacus_b200.Engine(lm.model, max_tokens=64 * 40, use_graphs=False, cache=form)
    c, d = bare.open(), bare.open()
    bare.step([(c, first[:150], [149]), (d, second[:5], [4])])
    bare.step([(c, first[150:200], [49]), (d, second[5:80], [74])])
    bare.step([(c, first[200:203], [2]), (d, second[80:81], [0])])
    for t in range(40):
        token = int(rng.integers(0, 515))
        x, y = engine.step([(a, [token], [0]), (b, [token], [0])]), bare.step([(c, [token], [0]), (d, [token], [0])])
        assert torch.equal(x, y), t
    # greedy generation in batches, the score of a text, as the 16-bit cache gives it to what 8 bits lose
    prompts = [first[:40], second[:33], first[60:64]]
    outs = lm.generate(prompts, max_new_tokens=20, temperature=0.0, stop_tokens=[])
    assert [len(o) for o in outs] == [20, 20, 20] and outs == lm.generate(prompts, max_new_tokens=20, temperature=0.0, stop_tokens=[])
    s, w = lm.score([first])[0], plain_lm.score([first])[0]
    assert np.abs(np.array(s.logprobs) - np.array(w.logprobs)).max() < 0.05 * float(want.abs().max())
    engine.check_status()


def test_first_pages_that_fall_and_models_that_have_other_mixers(tmp_path, ops):
    """kv8_read with a list that is not rising stays inside; an engine of another architecture, or in float32, refuses an 8-bit cache."""
    import abacus_b200
    import temetar_models
    run = Run(2, 1, 64, "int8", slots=3, pages=8)
    slots = [run.open() for _ in range(3)]
    batch = run.write(ops, [(s, 70) for s in slots], run.rows(210))
    k, v = (torch.full((6, 1, 64, 64), 7.0, device="cuda") for _ in range(2))
    for first in ([4, 2, 6, 0], [0, -5, 3, 2], [6, 5, 4, 3], [0, 100, 200, 300], [-3, -2, -1, 0]):
        ops.kv8_read(run.kv, batch, torch.tensor(first, dtype=torch.int32, device="cuda"), k, v)
    torch.cuda.synchronize()
    assert not any(ops.kernel_status(k.device).tolist())
    (tmp_path / "t").mkdir()
    (tmp_path / "q").mkdir()
    other = temetar_models.write_folder(tmp_path / "t", "P")[0]
    with pytest.raises(ValueError, match="8-bit"):
        abacus_b200.LM(other, cache="int8", max_tokens=256)
    folder = make_model_folder(tmp_path / "q", "D")
    with pytest.raises(ValueError, match="8-bit"):
        abacus_b200.LM(folder, dtype="float32", cache="int8", max_tokens=256)
    with pytest.raises(ValueError, match="int8 or e4m3"):
        abacus_b200.LM(folder, cache="fp8", max_tokens=256)


def test_windowed_layers_through_the_engine(tmp_path):
    """Full and windowed layers (rings of pages) of heads of 64 with the cache in 8 bits: decoded token by token far past the window, near the
    16-bit cache's logits."""
    import json
    import abacus_b200
    from abacus_b200.config import Qwen3Config
    from abacus_b200.weights import write_random_model
    raw = dict(hidden_size=128, intermediate_size=160, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=64,
               vocab_size=300, max_position_embeddings=512, rope_theta=10000.0, rms_norm_eps=1e-6, tie_word_embeddings=True,
               layer_types=["full_attention", "sliding_attention"], sliding_window=40, use_sliding_window=True,
               architectures=["Qwen3ForCausalLM"], model_type="qwen3")
    write_random_model(str(tmp_path), Qwen3Config.from_dict(raw), seed=4)
    rng = np.random.default_rng(2)
    tokens = rng.integers(0, 300, 330).tolist()
    logits = []
    for cache in (None, "int8"):
        lm = abacus_b200.LM(str(tmp_path), max_tokens=64 * 12, cache=cache)
        slot = lm.engine.open()
        got = [lm.engine.step([(slot, tokens[:130], [129])]).clone()]
        for t in tokens[130:]:
            got.append(lm.engine.step([(slot, [t], [0])]).clone())
        logits.append(torch.cat(got))
        if cache:
            with pytest.raises(Exception):
                lm.engine.step([(slot, tokens[:3], [2])])  # several tokens of a windowed layer go on with a sequence
    assert (logits[0] - logits[1]).abs().max() <= 0.05 * logits[0].abs().max()
