"""Log probabilities and the 8-bit cache, as cases that can be timed and compared.

A case is a dict of plain values; its "kind" names what a program does:

  logprobs  float32 or bfloat16 logits of some rows: the log probability of a given token, the entropy and the most likely
            tokens with theirs (ops.token_logprobs)
  product   the same without the most likely tokens, from the rows in front of the output matrix: the logits themselves are
            never kept (ops.gemm_tc_logprobs)
  keep      a step's keys and values go into a cache of 8 bits, whose sequences are then read back as pages
            (ops.kv8_write, ops.kv8_read)
  attend    a decode step, or one of a few tokens a sequence: the new keys and values go into the cache, the new rows attend
            to it (ops.kv8_write, ops.attention_kv8)

The cache holds blocks of 16 tokens of a sequence and kv head in 8 bits, q times the block's scale, with q a whole number
from -127 to 127 and the scale max|x| / 127 ("int8"), or q an e4m3 number and the scale max|x| / 448 ("e4m3"). A sequence's
last block, while it has fewer than 16 tokens, is held as it came. With `own` false everything here is in elementary torch
operations.
"""
import math

import torch

own = False

PAGE, BLOCK = 64, 16
TOP = {"int8": 127.0, "e4m3": 448.0}
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def _text(numbers):
    return ",".join(str(n) for n in numbers)


def _numbers(text):
    return [int(n) for n in text.split(",")]


def listed():
    return [
        # a decode step of eight users who each want the 20 most likely tokens beside the drawn one
        dict(name="logprobs_reply", kind="logprobs", rows=8, vocab=151936, dtype="float32", top=20, allowed=1.0),
        # a prompt of 512 tokens scored from its logits, with five alternatives at every place
        dict(name="logprobs_prompt", kind="logprobs", rows=512, vocab=151936, dtype="float32", top=5, allowed=1.0),
        # logits of 16 bits under a grammar that allows a twentieth of an odd vocabulary
        dict(name="logprobs_grammar", kind="logprobs", rows=200, vocab=50261, dtype="bfloat16", top=64, allowed=0.05),
        # a short answer scored under the 0.6B shape: the output matrix is read once
        dict(name="product_answer", kind="product", rows=37, width=1024, vocab=151936),
        # a prompt of 2,048 tokens under the 0.6B shape
        dict(name="product_prompt", kind="product", rows=2048, width=1024, vocab=151936),
        # a document under the 8B shape
        dict(name="product_document", kind="product", rows=4999, width=4096, vocab=151936),
        # unequal prompts of the 4B shape into a new cache
        dict(name="keep_prompts", kind="keep", starts="0,0,0,0,0,0", news="64,301,777,1024,1531,2048", heads=32, kv_heads=8,
             dim=128, form="int8"),
        # two long prompts that come in portions
        dict(name="keep_portions", kind="keep", starts="3584,1008", news="1001,512", heads=14, kv_heads=2, dim=64, form="e4m3"),
        # one user's next token under the 0.6B shape: launches and latency count
        dict(name="attend_one", kind="attend", starts="2175", news="1", heads=16, kv_heads=8, dim=128, form="int8", window=0),
        # 32 users of the 8B shape with contexts of 128 to 4,096
        dict(name="attend_users", kind="attend", starts=_text([127 + (3968 * i) // 31 for i in range(32)]), news=_text([1] * 32),
             heads=32, kv_heads=8, dim=128, form="int8", window=0),
        # two long documents
        dict(name="attend_documents", kind="attend", starts="131070,99999", news="1,1", heads=32, kv_heads=8, dim=128, form="e4m3",
             window=0),
        # four proposed tokens for each of 16 users, heads in groups of seven, a window
        dict(name="attend_proposals", kind="attend", starts=_text([304 + 16 * (37 * i % 200) + i % 13 for i in range(16)]),
             news=_text([4] * 16), heads=14, kv_heads=2, dim=64, form="int8", window=2000),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["logprobs", "product", "keep", "attend"])
    if kind == "logprobs":
        vocab = _log_int(rng, 1000, 262144)
        allowed = rng.choice([1.0, 1.0, 0.1])
        return dict(kind=kind, rows=_log_int(rng, 1, max(1, min(2000, 77_000_000 // vocab))), vocab=vocab,
                    dtype=rng.choice(["float32", "bfloat16"]), top=rng.choice([0, 1, 5, 20, 64]), allowed=allowed)
    if kind == "product":
        return dict(kind=kind, rows=_log_int(rng, 1, 4500), width=8 * _log_int(rng, 8, 512), vocab=_log_int(rng, 1000, 151936))
    dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 8, 16])
    form = rng.choice(["int8", "e4m3"])
    if kind == "keep":
        seqs = _log_int(rng, 1, 24)
        most = 48_000 // (seqs * kv_heads)
        return dict(kind=kind, starts=_text([BLOCK * rng.choice([0, 0, _log_int(rng, 1, max(1, most // BLOCK))]) for _ in range(seqs)]),
                    news=_text([_log_int(rng, 1, most) for _ in range(seqs)]), heads=heads, kv_heads=kv_heads, dim=dim, form=form)
    seqs = _log_int(rng, 1, 64)
    most = 1_600_000 // (seqs * kv_heads)
    new = rng.choice([1, 1, 1, 2, 4])
    starts = [_log_int(rng, 1, min(most, 131072)) - 1 for _ in range(seqs)]
    # (a step that closes a block and opens the next one is not the same step a second time; single tokens never are that)
    starts = [s if s % BLOCK + new <= BLOCK else s - BLOCK // 2 for s in starts]
    return dict(kind=kind, starts=_text(starts), news=_text([new] * seqs), heads=heads, kv_heads=kv_heads, dim=dim, form=form,
                window=rng.choice([0, 0, _log_int(rng, 16, 4096)]))


# ------------------------------------------------------------------ inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + 17)
    return g


def _quantized(x, form):
    """x [.., BLOCK, dim] -> (the numbers q as float32, the scales [..])."""
    x = x.to(torch.float32)
    most = x.abs().amax(dim=(-2, -1))
    scale = most / TOP[form]
    # (x * 127 is a float32 number whatever the bfloat16 x, so that the quotient is halfway between two steps where x is)
    q = x * TOP[form] / torch.where(most > 0, most, torch.ones_like(most))[..., None, None]
    if form == "int8":
        return q.round().clamp(-TOP[form], TOP[form]), scale
    return q.clamp(-TOP[form], TOP[form]).to(torch.float8_e4m3fn).to(torch.float32), scale


def _keys(shape, g):
    """Keys and values as a layer makes them: some channels are larger than others in every token."""
    x = torch.randn(shape, generator=g, device="cuda")
    return (x * (0.5 + torch.rand(shape[-1], generator=g, device="cuda") ** 4 * 6.0)).to(torch.bfloat16)


def _cache_state(case, g):
    """The cache before the step, the step's rows and what a program keeps for it."""
    starts, news = _numbers(case["starts"]), _numbers(case["news"])
    heads, kv_heads, dim, form = case["heads"], case["kv_heads"], case["dim"], case["form"]
    seqs = len(starts)
    of_seq = [-(-(s + n) // PAGE) for s, n in zip(starts, news)]
    pages = sum(of_seq) + 1
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(int(torch.randint(1 << 30, (1,), generator=g, device="cuda"))))
    table = torch.zeros((seqs, max(of_seq)), dtype=torch.int32)
    at = 0
    for i, n in enumerate(of_seq):
        table[i, :n] = order[at:at + n].to(torch.int32)
        at += n
    table = table.cuda()
    kind = torch.uint8 if form == "int8" else torch.float8_e4m3fn
    pool = [torch.zeros((pages, kv_heads, PAGE, dim), dtype=torch.uint8, device="cuda").view(kind) for _ in range(2)]
    scales = torch.zeros((pages, kv_heads, 2, PAGE // BLOCK), dtype=torch.float32, device="cuda")
    opened = torch.zeros((seqs, 2, kv_heads, BLOCK, dim), dtype=torch.bfloat16, device="cuda")
    for i, start in enumerate(starts):
        whole = start // BLOCK * BLOCK
        for j in range(2):
            for lo in range(0, whole, 32 * PAGE):  # some pages at a time
                hi = min(whole, lo + 32 * PAGE)
                x = _keys((kv_heads, hi - lo, dim), g)
                q, scale = _quantized(x.view(kv_heads, -1, BLOCK, dim), form)
                q = (q + 128.0).to(torch.uint8) if form == "int8" else q.to(torch.float8_e4m3fn).view(torch.uint8)
                at = table[i, lo // PAGE:-(-hi // PAGE)].long()
                blank = at.numel() * PAGE - (hi - lo)  # tokens of the last page that no whole block holds
                q = torch.nn.functional.pad(q.reshape(kv_heads, hi - lo, dim), (0, 0, 0, blank))
                scale = torch.nn.functional.pad(scale, (0, blank // BLOCK))
                pool[j].view(torch.uint8)[at] = q.view(kv_heads, -1, PAGE, dim).transpose(0, 1)
                scales[at, :, j] = scale.view(kv_heads, -1, PAGE // BLOCK).transpose(0, 1)
            if start > whole:
                opened[i, j, :, :start - whole] = _keys((kv_heads, start - whole, dim), g)
    rows = sum(news)
    qkv = torch.randn((rows, (heads + 2 * kv_heads) * dim), generator=g, device="cuda").to(torch.bfloat16)
    qkv[:, heads * dim:] = _keys((rows, 2 * kv_heads, dim), g).reshape(rows, -1)
    state = dict(case=case, starts=starts, news=news, table=table, k=pool[0], v=pool[1], scales=scales, open=opened, qkv=qkv,
                 first_page=[sum(of_seq[:i]) for i in range(seqs + 1)])
    state["out"] = torch.zeros((rows, heads * dim), dtype=torch.bfloat16, device="cuda")
    if case["kind"] == "keep":
        shape = (sum(of_seq), kv_heads, PAGE, dim)
        state["read"] = [torch.zeros(shape, dtype=torch.float32, device="cuda") for _ in range(2)]
    if own:
        from abacus_b200.cache import LayerKV8
        from abacus_b200.engine.batch import Sequence, StepBatch
        from abacus_b200.parts import Workspace
        state["ws"] = Workspace(qkv.device)
        state["cache"] = LayerKV8(pool[0], pool[1], scales, opened, table, table.shape[1])
        batch = StepBatch(rows, seqs, 1, "cuda")
        state["batch"] = batch.fill([Sequence(i, [0] * n, s, []) for i, (s, n) in enumerate(zip(starts, news))], exact=True)
        state["first_page_dev"] = torch.tensor(state["first_page"], dtype=torch.int32, device="cuda")
    return state


def prepare(case, seed):
    g = _generator(seed)
    if case["kind"] in ("keep", "attend"):
        return _cache_state(case, g)
    rows, vocab = case["rows"], case["vocab"]
    state = dict(case=case, logprob=torch.zeros(rows, device="cuda"), entropy=torch.zeros(rows, device="cuda"))
    if case["kind"] == "product":
        width = case["width"]
        state["x"] = torch.randn((rows, width), generator=g, device="cuda").to(torch.bfloat16)
        w = torch.empty((vocab, width), dtype=torch.bfloat16, device="cuda")
        for lo in range(0, vocab, 16384):
            w[lo:lo + 16384] = torch.randn((min(16384, vocab - lo), width), generator=g, device="cuda") * (2.0 / math.sqrt(width))
        state["w"] = w
        state["tokens"] = torch.randint(vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
        if own:
            from abacus_b200.parts import Workspace
            state["ws"] = Workspace(state["x"].device)
        return state
    # logits as a model gives them: a few tokens stand out, by more at some places than at others
    x = torch.randn((rows, vocab), generator=g, device="cuda") * 2.0
    likely = torch.randint(vocab, (rows, 40), generator=g, device="cuda")
    x.scatter_add_(1, likely, torch.rand((rows, 40), generator=g, device="cuda") * 14.0 * torch.rand((rows, 1), generator=g, device="cuda"))
    tokens = likely[:, 0].to(torch.int32)
    if case["allowed"] < 1.0:  # the same tokens are allowed in all rows, the given ones among them
        keep = torch.rand(vocab, generator=g, device="cuda") < case["allowed"]
        keep[:case["top"]] = True
        keep[tokens.long()] = True
        x[:, ~keep] = -math.inf
    state["logits"], state["tokens"] = x.to(TYPES[case["dtype"]]), tokens
    top = min(case["top"], vocab)
    state["top_ids"] = torch.zeros((rows, top), dtype=torch.int32, device="cuda") if top else None
    state["top_logprobs"] = torch.zeros((rows, top), device="cuda") if top else None
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    kind = state["case"]["kind"]
    if own:
        return _run_own(state, kind)
    if kind == "logprobs":
        return _logprobs(state["logits"].to(torch.float32), state["tokens"], state["case"]["top"])
    if kind == "product":
        logits = state["x"].to(torch.float32) @ state["w"].to(torch.float32).t()
        return _logprobs(logits, state["tokens"], 0)
    return _keep(state) if kind == "keep" else _attend(state)


def _run_own(state, kind):
    from abacus_b200.kernels import ops
    case = state["case"]
    if kind == "logprobs":
        ops.token_logprobs(state["logits"], state["tokens"], state["logprob"], entropy=state["entropy"], top_ids=state["top_ids"],
                           top_logprobs=state["top_logprobs"])
        out = dict(logprob=state["logprob"], entropy=state["entropy"])
        if case["top"]:
            out.update(ids=state["top_ids"], top=state["top_logprobs"])
        return out
    if kind == "product":
        ops.gemm_tc_logprobs(state["x"], state["w"], state["tokens"], state["logprob"], state["entropy"], state["ws"])
        return dict(logprob=state["logprob"], entropy=state["entropy"])
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    ops.kv8_write(state["qkv"], heads, kv_heads, dim, state["batch"], state["cache"])
    if kind == "keep":
        ops.kv8_read(state["cache"], state["batch"], state["first_page_dev"], *state["read"])
        return dict(k=state["read"][0], v=state["read"][1])
    ops.attention_kv8(state["qkv"], state["out"], heads, kv_heads, dim, dim ** -0.5, case["window"] or None, state["batch"],
                      state["cache"], state["ws"])
    return dict(out=state["out"])


def _logprobs(logits, tokens, top):
    most = logits.amax(dim=1, keepdim=True)
    d = logits - most
    e = torch.exp(d)
    total = e.sum(dim=1)
    log_total = torch.log(total)
    given = d.gather(1, tokens.long()[:, None])[:, 0]
    entropy = log_total - (e * torch.where(e > 0, d, torch.zeros_like(d))).sum(dim=1) / total
    out = dict(logprob=given - log_total, entropy=entropy)
    if top:
        values, ids = torch.sort(d, dim=1, descending=True, stable=True)
        out.update(ids=ids[:, :top].to(torch.int32).contiguous(), top=values[:, :top] - log_total[:, None])
    return out


def _held(state, i):
    """Keys and values of sequence i behind the step, [kv heads, tokens, dim] each: whole blocks as their 8 bits stand for."""
    case = state["case"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    start, new = state["starts"][i], state["news"][i]
    whole = start // BLOCK * BLOCK
    row = sum(state["news"][:i])
    got = []
    for j in range(2):
        pages = state["table"][i, :-(-whole // PAGE)].long()
        q = (state["k"], state["v"])[j].view(torch.uint8)[pages]
        q = q.to(torch.float32) - 128.0 if case["form"] == "int8" else q.view(torch.float8_e4m3fn).to(torch.float32)
        scale = state["scales"][pages, :, j].to(torch.float32)
        old = (q.view(-1, kv_heads, PAGE // BLOCK, BLOCK, dim) * scale[..., None, None]).permute(1, 0, 2, 3, 4).reshape(kv_heads, -1, dim)
        at = (heads + j * kv_heads) * dim
        rows = state["qkv"][row:row + new, at:at + kv_heads * dim].view(new, kv_heads, dim).permute(1, 0, 2)
        fresh = torch.cat([state["open"][i, j, :, :start - whole], rows], dim=1)
        closed = fresh.shape[1] // BLOCK * BLOCK
        q, scale = _quantized(fresh[:, :closed].reshape(kv_heads, -1, BLOCK, dim), case["form"])
        blocks = (q * scale[..., None, None]).reshape(kv_heads, closed, dim)
        got.append(torch.cat([old[:, :whole], blocks, fresh[:, closed:].to(torch.float32)], dim=1))
    return got


def _keep(state):
    kv_heads, dim = state["case"]["kv_heads"], state["case"]["dim"]
    out = [torch.zeros((state["first_page"][-1], kv_heads, PAGE, dim), dtype=torch.float32, device="cuda") for _ in range(2)]
    for i in range(len(state["starts"])):
        for pages, x in zip(out, _held(state, i)):
            n = state["first_page"][i + 1] - state["first_page"][i]
            x = torch.nn.functional.pad(x, (0, 0, 0, n * PAGE - x.shape[1]))
            pages[state["first_page"][i]:state["first_page"][i + 1]] = x.view(kv_heads, n, PAGE, dim).permute(1, 0, 2, 3)
    return dict(k=out[0], v=out[1])


def _attend(state):
    case = state["case"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    out, row = torch.empty_like(state["out"]), 0
    for i, (start, new) in enumerate(zip(state["starts"], state["news"])):
        k, v = _held(state, i)
        q = state["qkv"][row:row + new, :heads * dim].to(torch.float32).view(new, kv_heads, heads // kv_heads, dim)
        s = torch.einsum("nhgd,hkd->nhgk", q, k) * dim ** -0.5
        place = torch.arange(k.shape[1], device="cuda")
        mine = start + torch.arange(new, device="cuda")[:, None]
        seen = place <= mine
        if case["window"]:
            seen &= place > mine - case["window"]
        s = s.masked_fill(~seen[:, None, None], -math.inf)
        p = torch.exp(s - s.amax(dim=-1, keepdim=True))
        p = p / p.sum(dim=-1, keepdim=True)
        out[row:row + new] = torch.einsum("nhgk,hkd->nhgd", p, v).reshape(new, -1).to(torch.bfloat16)
        row += new
    return dict(out=out)


# ------------------------------------------------------------------ what a pass needs, and what it gives exactly
def work(case):
    if case["kind"] == "logprobs":
        n, vocab = case["rows"], case["vocab"]
        size = 4 if case["dtype"] == "float32" else 2
        return {"bytes": n * vocab * size + 4 * n * 3 + 8 * n * case["top"], "flops": 6 * n * vocab}
    if case["kind"] == "product":
        n, vocab, width = case["rows"], case["vocab"], case["width"]
        return {"bytes": 2 * (vocab + n) * width + 12 * n, "flops": 2 * n * vocab * width}
    starts, news = _numbers(case["starts"]), _numbers(case["news"])
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    token = 2 * kv_heads * dim  # values of a token's keys and values: a byte each in the cache, two in a step's rows
    if case["kind"] == "keep":
        tokens = sum(-(-(s + n) // PAGE) * PAGE for s, n in zip(starts, news))
        return {"bytes": 3 * token * sum(news) + token * sum(starts) + 4 * token * tokens, "flops": 4 * token * sum(news)}
    keys = read = 0
    for s, n in zip(starts, news):
        window = case["window"] or s + n
        keys += sum(min(s + j + 1, window) for j in range(n))
        read += min(s + n, window + n - 1)
    return {"bytes": token * (read + 2 * sum(news)) + 4 * heads * dim * sum(news), "flops": 4 * heads * dim * keys}


def exact(case, seed):
    state = prepare(case, seed)
    double = torch.float64
    if case["kind"] == "product":
        parts = [state["x"].to(double) @ w.to(double).t() for w in state["w"].split(16384)]
        return _exact_logprobs(torch.cat(parts, dim=1), state["tokens"], 0)
    if case["kind"] == "logprobs":
        return _exact_logprobs(state["logits"].to(double), state["tokens"], case["top"])
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "keep":
        pages = {"k": [], "v": []}
        for i in range(len(state["starts"])):
            for name, x in zip("kv", _exact_held(state, i)):
                n = state["first_page"][i + 1] - state["first_page"][i]
                whole = torch.zeros((kv_heads, n * PAGE, dim), dtype=double, device="cuda")
                whole[:, :x.shape[1]] = x
                pages[name] += [whole[:, PAGE * p:PAGE * (p + 1)] for p in range(n)]
        return {name: torch.stack(list_of) for name, list_of in pages.items()}
    out, row = torch.empty(state["out"].shape, dtype=double, device="cuda"), 0
    for i, (start, new) in enumerate(zip(state["starts"], state["news"])):
        k, v = _exact_held(state, i)
        for j in range(new):
            lo = max(0, start + j + 1 - case["window"]) if case["window"] else 0
            q = state["qkv"][row, :heads * dim].to(double).view(kv_heads, heads // kv_heads, dim)
            p = torch.softmax(q @ k[:, lo:start + j + 1].transpose(1, 2) / math.sqrt(dim), dim=-1)
            out[row] = (p @ v[:, lo:start + j + 1]).reshape(-1)
            row += 1
    return dict(out=out)


def _exact_held(state, i):
    """Keys and values of sequence i behind the step in 64 bits, [kv heads, tokens, dim] each, put together by token."""
    case, start, new = state["case"], state["starts"][i], state["news"][i]
    heads, kv_heads, dim, top = case["heads"], case["kv_heads"], case["dim"], TOP[case["form"]]
    token = torch.arange(start + new, device="cuda")
    first_new = sum(state["news"][:i])
    got = []
    for j, pool in enumerate((state["k"], state["v"])):
        x = torch.empty((start + new, kv_heads, dim), dtype=torch.float64, device="cuda")
        kept = token[:start // BLOCK * BLOCK]  # these were in 8 bits before the step
        page, place = state["table"][i].long()[kept // PAGE], kept % PAGE
        held = pool[page, :, place].to(torch.float64)
        if case["form"] == "int8":
            held = held - 128
        x[kept] = held * state["scales"][page, :, j, place // BLOCK].to(torch.float64)[..., None]
        x[kept.numel():start] = state["open"][i, j, :, :start - kept.numel()].transpose(0, 1).to(torch.float64)
        column = (heads + j * kv_heads) * dim
        x[start:] = state["qkv"][first_new:first_new + new, column:column + kv_heads * dim].reshape(new, kv_heads, dim).to(torch.float64)
        for lo in range(kept.numel(), (start + new) // BLOCK * BLOCK, BLOCK):
            block = x[lo:lo + BLOCK]
            most = block.abs().amax(dim=(0, 2))[:, None]
            step = most / top
            steps = block * top / torch.where(most == 0, torch.ones_like(most), most)
            steps = steps.round() if case["form"] == "int8" else steps.float().to(torch.float8_e4m3fn).to(torch.float64)
            x[lo:lo + BLOCK] = steps * step
        got.append(x.transpose(0, 1))
    return got


def _exact_logprobs(logits, tokens, top):
    logp = torch.log_softmax(logits, dim=1)
    p = torch.exp(logp)
    out = dict(logprob=logp[torch.arange(logp.shape[0], device="cuda"), tokens.long()],
               entropy=-torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(dim=1))
    if top:
        order = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :top]
        out.update(ids=order.to(torch.int32), top=logp.gather(1, order))
    return out
