"""The 8-bit cache at the steps between whole prompts and single tokens: several new tokens a sequence under windows and rings of pages."""
import pytest

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
