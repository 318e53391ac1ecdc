"""The 8-bit cache at the steps between whole prompts and single tokens: several new tokens a sequence under windows and rings of pages."""
import dataclasses

import numpy as np
import pytest
import torch

from helpers import make_model_folder
from test_kv8_gpu import Run, ops  # noqa: F401  (ops is a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form, dim, ring", [("int8", 64, True), ("e4m3", 128, True), ("int8", 128, False), ("e4m3", 64, False)])
@pytest.mark.parametrize("window", [1, 3, 15, 16, 64, 100])
def test_several_tokens_under_a_window(ops, window, form, dim, ring):  # noqa: F811
    """Steps of one to as many tokens as the ring allows (of up to 114 over a table with all pages), beginning and ending anywhere in
    a block: each row's first visible key lies inside a block of earlier steps, one that the step closes, or the open one. One
    token more than the ring allows is refused."""
    run = Run(6, 2, dim, form, slots=2, pages=30, window=window if ring else None, max_context=900)
    run.window = window
    most = run.kv.ring_pages * 64 - window + 1 if ring else 114
    a, b = run.open(), run.open()
    run.write(ops, [(a, 10), (b, 37)], run.rows(47))
    for news in ([(a, most), (b, 1)], [(a, 5), (b, most)], [(a, 1), (b, 3)], [(b, most - 7), (a, 17)], [(a, most)], [(b, 16), (a, 2)]):
        qkv = run.rows(sum(n for _, n in news))
        run.attend(ops, run.write(ops, news, qkv), qkv)
    if ring:
        batch = run.batch([(a, most + 1)])
        qkv = run.rows(most + 1).cuda()
        with pytest.raises(ops.KernelRefused, match="ring"):
            ops.attention_kv8(qkv, qkv.new_zeros((most + 1, 6 * dim)), 6, 2, dim, 0.125, window, batch, run.kv, run.ws)


def model_of(folder, schedule=None):
    """The bfloat16 model of a folder, with its layers in another order."""
    from abacus_b200.config import load_config
    from abacus_b200.models import Model
    from abacus_b200.weights import load_folder
    arch, cfg = load_config(folder)
    spec = cfg.to_spec() if schedule is None else dataclasses.replace(cfg.to_spec(), schedule=schedule)
    tensors = load_folder(folder, lambda names: arch.tensor_names(spec, names))
    return Model(spec, arch.layout(spec), tensors, torch.bfloat16, torch.device("cuda", 0))


def test_prompts_of_a_layer_that_reads_anothers_cache_again_and_again(tmp_path):
    """Prompt steps of one shape, the lengths and slots others each time: an engine that captures steps gives what one without graphs
    gives (the pages that the second layer reads back are this step's, not an earlier one's)."""
    from abacus_b200.config import ScheduleEntry
    from abacus_b200.engine import Engine
    model = model_of(make_model_folder(tmp_path, "D"), (ScheduleEntry(0), ScheduleEntry(1, source=0), ScheduleEntry(1)))
    engines = [Engine(model, max_tokens=64 * 20, use_graphs=graphs, cache="int8") for graphs in (True, False)]
    rng = np.random.default_rng(3)
    for lengths in ((100, 150), (140, 110), (90, 160), (155, 95), (150, 100)):
        prompts = [rng.integers(0, 515, n).tolist() for n in lengths]
        got = []
        for e in engines:
            slots = [e.open() for _ in prompts]
            logits = e.step([(s, p, [len(p) - 1]) for s, p in zip(slots, prompts)]).clone()
            logits = torch.cat([logits, e.step([(s, [7], [0]) for s in slots])])
            for s in slots[::-1]:
                e.close(s)
            e.check_status()
            got.append(logits)
        assert torch.equal(*got), lengths


def test_what_is_not_there_is_reported_after_the_launch_before(ops):  # noqa: F811
    """The status bits of a bad page or slot come when the launch before has ended, so one that sets the status to zero does not take
    them away; rows of a good slot are as they were."""
    from abacus_b200.engine.batch import Sequence, StepBatch
    run = Run(2, 1, 64, "int8", slots=3, pages=6)
    a, b = run.open(), run.open()
    run.write(ops, [(a, 70), (b, 30)], run.rows(100))
    qkv = run.rows(2).cuda()
    status = ops.kernel_status(qkv.device)
    out, good = torch.zeros((2, 128), dtype=torch.bfloat16, device="cuda"), torch.zeros((2, 128), dtype=torch.bfloat16, device="cuda")
    batch = StepBatch(2, 2, 1, "cuda").fill([Sequence(b, [0], 29, []), Sequence(a, [0], 69, [])], exact=True)
    ops.attention_kv8(qkv, good, 2, 1, 64, 0.125, None, batch, run.kv, run.ws)
    lost = torch.zeros(1 << 22, dtype=torch.int32, device="cuda")
    for slot, bad_page, bit in ((7, False, 4), (-1, False, 4), (a, True, 2)):
        batch = StepBatch(2, 2, 1, "cuda").fill([Sequence(b, [0], 29, []), Sequence(slot, [0], 69, [])], exact=True)
        table = run.kv.page_table.clone()
        if bad_page:
            run.kv.page_table[a, 0] = 1000
        for _ in range(20):
            lost.zero_()  # (a launch of a while)
            status.zero_()
            ops.attention_kv8(qkv, out, 2, 1, 64, 0.125, None, batch, run.kv, run.ws)
            assert status.tolist()[2] == bit and torch.equal(out[0], good[0])
        run.kv.page_table.copy_(table)
    status.zero_()


@pytest.mark.parametrize("ring", [True, False])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_open_tokens_before_the_window_may_hold_anything(ops, ring, bad):  # noqa: F811
    """Keys and values that are not finite, in a sequence's open block but before a row's window: nothing of them reaches the row."""
    run = Run(4, 2, 64, "int8", slots=2, pages=6, window=5 if ring else None, max_context=200)
    run.window = 5
    a, b = run.open(), run.open()
    spoilt = run.rows(23)
    spoilt[:4, 4 * 64:], spoilt[22, 4 * 64:] = bad, bad  # tokens 0 to 3 of a, token 18 of b
    run.write(ops, [(a, 4), (b, 19)], spoilt)
    run.write(ops, [(a, 4), (b, 4)], run.rows(8))
    for slot in (a, b):  # (the formula takes them as zeros, which no row sees either)
        run.brought[slot] = [torch.nan_to_num(x, 0.0, 0.0, 0.0) for x in run.brought[slot]]
    for _ in range(3):
        qkv = run.rows(2)
        run.attend(ops, run.write(ops, [(a, 1), (b, 1)], qkv), qkv)


@pytest.mark.parametrize("form", ["int8", "e4m3"])
def test_attention_right_behind_a_write_of_another_step(ops, form):  # noqa: F811
    """Rows that attend to what a larger step's kv8_write has just put into the cache: the last tokens of a long prompt as a step of their
    own, and a decode step moved on by the device. Such calls wait for the launch before (the same step's kv8_write lets them read ahead)."""
    from abacus_b200.engine.batch import Sequence, StepBatch
    run = Run(8, 2, 128, form, slots=6, pages=400, max_context=1 << 13)
    for new in (4, 1):
        slots = [run.open() for _ in range(3)]
        lengths = [8000, 5003, 7001]
        qkv = run.rows(sum(lengths))
        tail = StepBatch(3 * new, 3, 1, "cuda").fill([Sequence(s, [0] * new, n - new, []) for s, n in zip(slots, lengths)], exact=True)
        ends = np.cumsum(lengths)
        rows = torch.cat([qkv[e - new:e] for e in ends])
        on_gpu, out, whole = rows.cuda(), torch.zeros((3 * new, 8 * 128), dtype=torch.bfloat16, device="cuda"), qkv.cuda()
        batch = run.batch(list(zip(slots, lengths)))
        torch.cuda.synchronize()
        ops.kv8_write(whole, 8, 2, 128, batch, run.kv)
        ops.attention_kv8(on_gpu, out, 8, 2, 128, 128 ** -0.5, None, tail, run.kv, run.ws)
        assert batch.kv8_written is run.kv and tail.kv8_written is None
        torch.cuda.synchronize()
        again = torch.zeros_like(out)
        ops.attention_kv8(on_gpu, again, 8, 2, 128, 128 ** -0.5, None, tail, run.kv, run.ws)
        assert torch.equal(out, again)
        for s in slots:
            run.cache.close_slot(s)
    one = StepBatch(1, 1, 1, "cuda").fill([Sequence(run.open(), [0], 0, [])], exact=True)
    run.cache.reserve(one.sequences[0].slot, 8)
    ops.kv8_write(rows[:1].cuda(), 8, 2, 128, one, run.kv)
    assert one.kv8_written is run.kv and one.advance_on_device().kv8_written is None


def windowed_folder(tmp_path):
    """A model folder of three layers of heads of 64, the second windowed."""
    import os
    from abacus_b200.config import Qwen3Config
    from abacus_b200.weights import write_random_model
    raw = dict(hidden_size=128, intermediate_size=160, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=2, head_dim=64,
               vocab_size=300, max_position_embeddings=512, rope_theta=10000.0, rms_norm_eps=1e-6, tie_word_embeddings=True,
               layer_types=["full_attention", "sliding_attention", "full_attention"], sliding_window=40, use_sliding_window=True,
               architectures=["Qwen3ForCausalLM"], model_type="qwen3")
    return write_random_model(os.path.join(str(tmp_path), "w"), Qwen3Config.from_dict(raw), seed=4)


def test_a_refused_step_leaves_the_cache_as_it_was(tmp_path, ops):  # noqa: F811
    """Several tokens that go on with a windowed sequence are refused before the layers in front have written: the sequence goes on as if
    nobody had asked (the refused tokens would have closed its open block and begun another)."""
    import abacus_b200
    lm = abacus_b200.LM(windowed_folder(tmp_path), max_tokens=64 * 12, cache="int8")
    rng = np.random.default_rng(2)
    tokens, engine, got = rng.integers(0, 300, 60).tolist(), lm.engine, []
    for asks in (False, True):
        slot = engine.open()
        rows = [engine.step([(slot, tokens[:13], [12])]).clone()]
        if asks:
            with pytest.raises(ops.KernelRefused, match="windowed"):
                engine.step([(slot, tokens[:5], [4])])
            with pytest.raises(ops.KernelRefused, match="windowed"):
                engine.score([(slot, tokens[:5], [4])], [1])
        rows += [engine.step([(slot, [t], [0])]).clone() for t in tokens[13:]]
        got.append(torch.cat(rows))
        engine.close(slot)
    assert torch.equal(*got)


@pytest.mark.parametrize("borrows", [False, True])
@pytest.mark.parametrize("form", ["int8", "e4m3"])
def test_a_sequence_goes_the_same_way_whatever_is_beside_it(tmp_path, monkeypatch, form, borrows):
    """A whole prompt, a short one, a portion, a few tokens and a single one in one step give the bits that they give in steps of their own
    (a prompt attends to its keys as they came beside a sequence that goes on, too), logits and scores; portions that are more context than is read
    back at a time go one after the other; last_batch holds the step's sequences."""
    from abacus_b200.config import ScheduleEntry
    from abacus_b200.engine import Engine, engine as module
    monkeypatch.setattr(module, "READ_BACK_TOKENS", 150)
    schedule = (ScheduleEntry(0), ScheduleEntry(1, source=0), ScheduleEntry(1)) if borrows else None
    model = model_of(make_model_folder(tmp_path, "D"), schedule)
    rng = np.random.default_rng(5)
    before, news = [40, 0, 90, 77, 70], [30, 50, 20, 3, 25]
    if borrows:
        before, news = before + [0], news + [6]
    texts = [rng.integers(0, 515, b + n).tolist() for b, n in zip(before, news)]
    for score in (False, True):
        got = []
        for together in (True, False):
            engine = Engine(model, max_tokens=64 * 20, use_graphs=False, cache=form)
            slots = [engine.open() for _ in texts]
            for slot, text, n in zip(slots, texts, before):
                if n:
                    engine.step([(slot, text[:n], [])])
            entries = [(slot, text[n:], [0, len(text) - n - 1] if n != 77 else [1]) for slot, text, n in zip(slots, texts, before)]
            steps = [entries] if together else [[e] for e in entries]
            if score:
                parts = [engine.score(step, [int(t) for _, text, want in step for t in text[:len(want)]], top=3) for step in steps]
                got.append([torch.cat([p[i] for p in parts]) for i in range(4)])
            else:
                got.append([torch.cat([engine.step(step).clone() for step in steps])])
            if together:
                assert [s.slot for s in engine.last_batch.sequences] == slots and engine.last_batch.n_rows == sum(news)
            assert [engine.length(s) for s in slots] == [len(t) for t in texts]
            engine.check_status()
        assert all(torch.equal(x, y) for x, y in zip(*got))


@pytest.mark.parametrize("form", ["int8", "e4m3"])
@pytest.mark.parametrize("windowed", [False, True])
def test_a_score_reads_the_8_bit_cache(tmp_path, form, windowed):
    """LM.score(from_cache=True): the numbers of texts whose tokens go on with their first one (single tokens where a layer is windowed), which
    are not those of whole texts, the default's. Texts of one token, of two, unequal ones. A 16-bit cache has one kind of score."""
    import abacus_b200
    folder = windowed_folder(tmp_path) if windowed else make_model_folder(tmp_path, "D")
    lm = abacus_b200.LM(folder, max_tokens=64 * 20, cache=form)
    rng = np.random.default_rng(8)
    texts = [rng.integers(0, 300, n).tolist() for n in (1, 2, 75, 40)]
    engine = lm.engine

    def by_hand(cuts):
        slots, rows = [engine.open() for _ in texts], [[] for _ in texts]
        for lo, hi in zip(cuts, cuts[1:]):
            here = [i for i, t in enumerate(texts) if len(t) > lo]
            wants = [list(range(min(hi, len(texts[i]) - 1) - lo)) for i in here]
            got = engine.score([(slots[i], texts[i][lo:hi], w) for i, w in zip(here, wants)],
                               [texts[i][lo + 1 + p] for i, w in zip(here, wants) for p in w], top=2)
            at = 0
            for i, w in zip(here, wants):
                rows[i] += zip(*(x[at:at + len(w)].tolist() for x in got))
                at += len(w)
        for s in slots:
            engine.close(s)
        return rows

    for from_cache, cuts in ((False, (0, 75)), (True, range(76) if windowed else (0, 1, 75))):
        scores = lm.score(texts, top=2, from_cache=from_cache)
        for s, text, rows in zip(scores, texts, by_hand(list(cuts))):
            assert s.tokens == text and len(s.logprobs) == len(s.entropies) == len(s.top) == len(text) - 1
            assert [(p, h, [i for i, _ in t], [v for _, v in t]) for p, h, t in zip(s.logprobs, s.entropies, s.top)] == rows
    assert lm.score(texts)[2].logprobs == lm.score(texts, from_cache=False)[2].logprobs != lm.score(texts, from_cache=True)[2].logprobs
    assert lm.engine.cache.free_pages == lm.engine.cache.n_pages
    plain = abacus_b200.LM(folder, max_tokens=64 * 20)
    assert plain.score(texts, from_cache=True)[2].logprobs == plain.score(texts)[2].logprobs


@pytest.mark.parametrize("form", ["int8", "e4m3"])
def test_every_quotient_of_two_mantissas(ops, form):  # noqa: F811
    """Blocks whose largest number has every mantissa M of 8 bits, with every other mantissa at eight sizes below it, of both signs: each
    is rounded as the exact quotient is (254 / 255 comes within 2^-16 of a tie, 127 x 2^-s / 255 and others are ties)."""
    run = Run(1, 1, 64, form, slots=1, pages=40)
    a = run.open()
    qkv = torch.zeros((128 * 16, 3 * 64))
    x = torch.arange(128, 256).float()[:, None] * 2.0 ** -torch.arange(8).float()  # [mantissas, sizes]
    for i, m in enumerate(range(128, 256)):
        block = torch.where(x <= m, x, torch.zeros(())).reshape(-1) * (1 - 2 * (torch.arange(1024) % 3 == 0).float())
        block[0] = m
        qkv[16 * i:16 * i + 16, 64:] = block.view(16, 64).repeat(1, 2)
    qkv = qkv.to(torch.bfloat16)
    assert (qkv[127 * 16:, 64:].float().abs() == 254).any() and float(qkv.abs().max()) == 255
    run.check(ops, run.write(ops, [(a, 128 * 16)], qkv))


def test_a_mixed_step_of_a_windowed_model_and_one_that_asks_for_what_is_not_there(tmp_path):
    """Whole prompts and single tokens of a windowed model in one step give the bits of steps apart; a wanted place beyond a sequence's
    tokens is refused with no sequence moved, whichever pass it would have been in."""
    from abacus_b200.engine import Engine
    model = model_of(windowed_folder(tmp_path))
    rng = np.random.default_rng(6)
    first, second, third = (rng.integers(0, 300, n).tolist() for n in (61, 83, 9))
    got = []
    for together in (True, False):
        engine = Engine(model, max_tokens=64 * 12, use_graphs=False, cache="e4m3")
        a, b, c = (engine.open() for _ in range(3))
        engine.step([(a, first, []), (c, third, [])])
        entries = [(a, [5], [0]), (b, second, [3, 82])]
        if together:
            for bad in (1, -1):
                with pytest.raises(ValueError, match="wanted place"):
                    engine.step([(a, [5], [0]), (b, second, [bad * 83])])
                with pytest.raises(ValueError, match="wanted place"):
                    engine.step([(a, [5], [bad]), (b, second, [0])])
            assert [engine.length(s) for s in (a, b, c)] == [61, 0, 9]
        steps = [entries] if together else [[e] for e in entries]
        rows = [engine.step(step).clone() for step in steps]
        rows.append(engine.step([(a, [7], [0])]).clone())
        rows.append(engine.step([(b, [8], [0])]).clone())
        got.append(torch.cat(rows))
        engine.check_status()
    assert torch.equal(*got)
