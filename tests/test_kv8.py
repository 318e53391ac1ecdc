"""The 8-bit cache's bookkeeping, what is refused before anything runs, and the command line's options: no GPU."""
import pytest
import torch

from abacus_b200 import cli
from abacus_b200.cache import CacheNeed, LayerKV8, SequenceCache


def layer(pages=3, heads=2, dim=64, slots=2, kind=torch.uint8):
    return dict(k=torch.zeros((pages, heads, 64, dim), dtype=torch.uint8).view(kind), v=torch.zeros((pages, heads, 64, dim), dtype=torch.uint8).view(kind),
                scales=torch.zeros((pages, heads, 2, 4)), open=torch.zeros((slots, 2, heads, 16, dim), dtype=torch.bfloat16),
                page_table=torch.zeros((slots, 5), dtype=torch.int32), table_width=5)


def test_a_layer_knows_its_form_and_room():
    assert LayerKV8(**layer()).form == "int8" and LayerKV8(**layer(kind=torch.float8_e4m3fn)).form == "e4m3"
    kv = LayerKV8(**layer(pages=7, heads=3, dim=128, slots=4))
    assert (kv.n_pages, kv.n_kv_heads, kv.head_dim, kv.n_slots, kv.room) == (7, 3, 128, 4, 5 * 64)
    assert LayerKV8(**layer(), ring_pages=2, window=20).room is None


@pytest.mark.parametrize("change", [
    dict(k=torch.zeros((3, 2, 64, 64), dtype=torch.int8)), dict(k=torch.zeros((3, 2, 32, 64), dtype=torch.uint8)),
    dict(v=torch.zeros((4, 2, 64, 64), dtype=torch.uint8)), dict(v=torch.zeros((3, 2, 64, 64), dtype=torch.uint8).view(torch.float8_e4m3fn)),
    dict(scales=torch.zeros((3, 2, 2, 4), dtype=torch.float64)), dict(scales=torch.zeros((3, 2, 4, 2))),
    dict(open=torch.zeros((2, 2, 2, 16, 64))), dict(page_table=torch.zeros((2, 4), dtype=torch.int32)),
    dict(page_table=torch.zeros((2, 5), dtype=torch.int64)), dict(k=torch.zeros((3, 2, 64, 128), dtype=torch.uint8)[..., ::2]),
    dict(pinned_pages=1), dict(tokens_per_page=32), dict(values_in_keys=True)])
def test_a_layer_that_does_not_fit_together_is_refused(change):
    with pytest.raises(ValueError):
        LayerKV8(**{**layer(), **change})


@pytest.mark.parametrize("form", ["int8", "e4m3"])
def test_a_sequence_cache_in_8_bits(form):
    needs = [CacheNeed(2, 64), CacheNeed(2, 64, window=24), CacheNeed(2, 64), None]
    cache = SequenceCache(needs, [None, None, None, 0], 640, torch.bfloat16, "cpu", max_slots=3, form=form)
    kv = cache.views[0].kv
    assert isinstance(kv, LayerKV8) and kv.form == form and cache.views[3].kv.k.data_ptr() == kv.k.data_ptr()
    assert cache.views[2].kv.k.data_ptr() != kv.k.data_ptr() and cache.views[2].kv.open.data_ptr() != kv.open.data_ptr()
    assert cache.views[1].kv.ring_pages == 2 and cache.views[1].kv.window == 24
    a = cache.open_slot()
    cache.reserve(a, 130)
    assert kv.page_table[a, :3].tolist() == cache.groups[0].book.of_slot[a]
    wide = SequenceCache(needs, [None, None, None, 0], 640, torch.bfloat16, "cpu", max_slots=3)
    opened = sum(g.open.numel() * 2 for g in cache.groups)
    assert cache.bytes() - opened < 0.52 * wide.bytes()


def test_what_an_8_bit_cache_does_not_hold_is_refused():
    for need in (CacheNeed(2, 48), CacheNeed(2, 64, v_head_dim=32), CacheNeed(1, 64, values_in_keys=True, v_head_dim=32),
                 CacheNeed(2, 64, window=20, keep_first=4)):
        with pytest.raises(ValueError, match="8-bit"):
            SequenceCache([need], [None], 640, torch.bfloat16, "cpu", form="int8")
    with pytest.raises(ValueError, match="int4"):
        SequenceCache([CacheNeed(2, 64)], [None], 640, torch.bfloat16, "cpu", form="int4")


def test_kernels_refuse_tensors_that_are_not_on_the_gpu():
    from abacus_b200.kernels import ops
    x, t = torch.zeros((2, 5)), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ops.KernelError, match="not on the GPU"):
        ops.token_logprobs(x, t, torch.zeros(2))
    with pytest.raises(ops.KernelError, match="not on the GPU"):
        ops.gemm_tc_logprobs(torch.zeros((2, 8), dtype=torch.bfloat16), torch.zeros((5, 8), dtype=torch.bfloat16), t, torch.zeros(2), None, None)


def test_command_line_options():
    o = cli.parse(["m", "--score", "a text", "--kv8", "e4m3"])
    assert o.score == "a text" and o.kv8 == "e4m3"
    assert cli.parse(["m"]).score is None and cli.parse(["m"]).kv8 is None
    with pytest.raises(cli.UsageError, match="int8 and e4m3"):
        cli.parse(["m", "--kv8", "int4"])
