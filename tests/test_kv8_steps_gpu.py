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
