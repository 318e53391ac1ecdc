"""Keys and values in 8 bits, with a scale for each block of 16 tokens and kv head.

A whole block of a sequence and kv head is kept as 8-bit numbers in the pages that the 16-bit cache would use too, and a
float32 scale for its keys and one for its values. "int8": whole numbers from -127 to 127, stored as q + 128, the scale
max|x| / 127. "e4m3": e4m3 numbers, the scale max|x| / 448. The last block of a sequence, until it has 16 tokens, lies as it came
(bfloat16) in the slot's open block: nothing is rounded twice, and a scale is made once, from the whole block.
csrc/kv8.cu makes and reads them, csrc/attention_kv8.cu attends to them.
"""
from dataclasses import dataclass
from typing import Optional

import torch

from ..kernels import guards

PAGE, BLOCK = 64, 16
FORMS = {"int8": torch.uint8, "e4m3": torch.float8_e4m3fn}


@dataclass(frozen=True)
class LayerKV8:
    """What the kernels need to find a sequence's keys and values of one schedule entry in an 8-bit cache. The tensors are looked at
    once, here: their addresses and sizes go to every call."""
    k: torch.Tensor       # uint8 ("int8") or float8_e4m3fn ("e4m3") [pages, kv heads, 64, head_dim]
    v: torch.Tensor
    scales: torch.Tensor  # float32 [pages, kv heads, 2 (keys, values), 4 blocks of the page]
    open: torch.Tensor    # bfloat16 [slots, 2 (keys, values), kv heads, 16, head_dim]
    page_table: torch.Tensor  # int32 [slots, table_width]
    table_width: int
    ring_pages: int = 0
    window: Optional[int] = None
    tokens_per_page: int = PAGE
    pinned_pages: int = 0
    values_in_keys: bool = False

    def __post_init__(self):
        pages, heads, tokens, dim = self.k.shape
        if self.k.dtype not in FORMS.values():
            raise ValueError(f"8-bit keys are uint8 (q + 128) or float8_e4m3fn, not {self.k.dtype}")
        if tokens != PAGE or self.tokens_per_page != PAGE or self.pinned_pages or self.values_in_keys:
            raise ValueError(f"pages of an 8-bit cache hold {PAGE} tokens, none of them pinned, values apart from keys")
        wanted = {"v": (self.v, self.k.dtype, (pages, heads, tokens, dim)),
                  "scales": (self.scales, torch.float32, (pages, heads, 2, PAGE // BLOCK)),
                  "open": (self.open, torch.bfloat16, (self.open.shape[0], 2, heads, BLOCK, dim)),
                  "page_table": (self.page_table, torch.int32, (self.open.shape[0], self.table_width)),
                  "k": (self.k, self.k.dtype, (pages, heads, tokens, dim))}
        for name, (t, dtype, shape) in wanted.items():
            if t.dtype != dtype or tuple(t.shape) != shape or not t.is_contiguous():
                raise ValueError(f"{name} of an 8-bit cache is contiguous, {dtype} {shape}; got {t.dtype} {tuple(t.shape)}")
            if t.device != self.k.device:
                raise ValueError(f"{name} of an 8-bit cache is on {t.device}, its keys on {self.k.device}")

        known = dict(form="int8" if self.k.dtype == torch.uint8 else "e4m3", n_pages=pages, n_kv_heads=heads, head_dim=dim,
                     n_slots=self.open.shape[0], device_index=self.k.get_device(), record=None,  # (ops.Kv8Cache, at the first call)
                     room=None if self.ring_pages else self.table_width * PAGE)
        for name, value in known.items():
            object.__setattr__(self, name, value)


def pools(n_entries, n_pages, n_slots, n_kv_heads, head_dim, form, device):
    """(k, v, scales, open) of n_entries schedule entries, zeroed, each with the entries as its first dimension."""
    if form not in FORMS:
        raise ValueError(f"8-bit cache {form!r}: the forms are {', '.join(FORMS)}")
    pages = (n_entries, n_pages, n_kv_heads)
    k, v = (_zeros(pages + (PAGE, head_dim), form, device, f"8-bit cache {what}") for what in ("keys", "values"))
    scales = guards.zeros(pages + (2, PAGE // BLOCK), torch.float32, device, what="scales of the 8-bit cache")
    opened = guards.zeros((n_entries, n_slots, 2, n_kv_heads, BLOCK, head_dim), torch.bfloat16, device, what="open blocks of the 8-bit cache")
    return k, v, scales, opened


def _zeros(shape, form, device, what):
    plain = guards.zeros(shape, torch.uint8, device, what=what)
    out = plain.view(FORMS[form])
    if out is not plain and hasattr(plain, "guarded_allocation"):
        out.guarded_allocation = plain.guarded_allocation  # (the guards live as long as the tensor handed out)
    return out
