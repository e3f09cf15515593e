"""A serving step around a model as cases that can be timed and compared: which blocks of a paged cache requests hold, where
their new tokens go, and which ids are drawn from the logits.

``op`` says which entry point of ``gputok_b200.Tokenizer`` a case goes through:

  tables    block_tables   requests that grow take blocks of the cache from a queue, those that shrink give them back
  slots     slot_map       place in the cache, position and request of every new token
  sample    sample         an id per row of logits with temperature, top-k, top-p and min-p, from a given random number

With ``own`` false ``run`` computes them in elementary torch operations instead; weights and their sums in 64 bits, since an id
is a comparison of sums of many numbers with each other.

Logits are normal with a head of likely ids, whose lead differs from row to row: a model is sure of some tokens and not of others.
"""
from __future__ import annotations

import functools
import math
import os
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
GPT2 = 50257  # GPT-2's ids: 256 bytes, 50 000 merges, end of text
HEAD = 64     # ids per row that lead the others


def _sample(n, vocab, type_, temperature=1.0, top_k=0, top_p=0.0, min_p=0.0, mixed=False, pitch=0, masked=False, padded=False):
    """0 for a limit that is off; mixed: every row has limits of its own, as far as they are on."""
    return {"op": "sample", "n": n, "vocab": vocab, "type": type_, "temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p,
            "mixed": mixed, "pitch": pitch or vocab, "masked": masked, "padded": padded}


def _tables(n, block, longest, kind):
    return {"op": "tables", "n": n, "block": block, "longest": longest, "kind": kind}


def _slots(n, block, longest, kind, tokens):
    return {"op": "slots", "n": n, "block": block, "longest": longest, "kind": kind, "tokens": tokens}


def listed():
    return [
        # the next token of one running text, with the usual limits
        dict(_sample(1, GPT2, "bf16", 0.8, 50, 0.95), name="sample one token"),
        # the most likely ids of a batch, as evaluations take them
        dict(_sample(512, GPT2, "bf16", 0.0), name="sample greedily"),
        # a server's batch: every request has limits of its own, some rows of the batch are empty, the vocabulary is padded
        dict(_sample(256, GPT2, "f32", 0.9, 40, 0.9, 0.05, True, 50304, False, True), name="sample for many users"),
        # a nucleus of a large vocabulary, fewer rows than the GPU has SMs
        dict(_sample(64, 131072, "f32", 0.7, 0, 0.95), name="sample a nucleus"),
        # flat distributions: a warm temperature and a nucleus of thousands of ids; part of the ids is masked; odd sizes
        dict(_sample(333, 32003, "f16", 1.3, 0, 0.99, 0.0, False, 0, True), name="sample wide nuclei"),
        # rollouts for reinforcement learning: the model's own distribution, no limits
        dict(_sample(1024, 131072, "bf16", 1.0), name="sample rollouts"),
        # a decoding step: most requests grow by a token, some end, some begin
        dict(_tables(256, 16, 4096, "step"), name="tables, a decoding step"),
        # many requests of which half are replaced by others
        dict(_tables(8192, 16, 8192, "replace"), name="tables, requests come and go"),
        # a decoding step's slots: one token per request
        dict(_slots(256, 16, 4096, "step", 256), name="slots, a decoding step"),
        # prompts in pieces and running requests in one batch of fixed size, blocks of an odd size
        dict(_slots(700, 24, 8192, "mixed", 8192), name="slots, prompts in pieces"),
        # long prompts of a batch at once
        dict(_slots(512, 64, 131072, "prompts", 1 << 20), name="slots, long prompts"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["sample", "sample", "tables", "slots"])
    if op == "sample":
        vocab = GPT2 if rng.random() < 0.3 else _log(rng, 257, 131072)
        n = min(_log(rng, 1, 1024), (1 << 26) // vocab)
        pitch = (vocab + 63) // 64 * 64 if rng.random() < 0.5 else vocab
        return _sample(n, vocab, rng.choice(sorted(TYPES)), rng.choice([0.0, round(rng.uniform(0.3, 1.5), 3), round(rng.uniform(0.3, 1.5), 3)]),
                       _log(rng, 2, 1000) if rng.random() < 0.5 else 0, round(1 - 10 ** rng.uniform(-3, -0.3), 4) if rng.random() < 0.5 else 0.0,
                       round(10 ** rng.uniform(-3, -0.5), 4) if rng.random() < 0.3 else 0.0, rng.random() < 0.4, pitch, rng.random() < 0.3,
                       rng.random() < 0.3)
    block = rng.choice([8, 16, 24, 32, 64, 100, 128, 256])
    if op == "tables":
        return _tables(_log(rng, 1, 8192), block, _log(rng, 64, 8192), rng.choice(["step", "replace"]))
    n = _log(rng, 1, 8192)
    kind = rng.choice(["step", "mixed", "prompts"])
    tokens = n if kind == "step" else _log(rng, n, 1 << 20)
    longest = max(_log(rng, 256, 16384), 2 * tokens // n) if n < 2048 else 4096
    return _slots(n, block, min(longest, (1 << 23) // n * block), kind, tokens)


@functools.lru_cache(maxsize=None)
def _tokenizer_on(device, stream):
    for p in (ROOT, os.path.join(ROOT, "gpu-tokenizer_b200")):
        if p not in sys.path:
            sys.path.insert(0, p)
    import gputok_b200

    tok = gputok_b200.Tokenizer(os.path.join(ROOT, "tests", "golden", "gpt2_merges.txt"), device=device)
    tok.set_stream(stream)
    return tok


def _tokenizer():
    """The handle for torch's current device and stream, which a state's inputs are made on and its passes run on."""
    return _tokenizer_on(torch.cuda.current_device(), torch.cuda.current_stream().cuda_stream)


# ---------------------------------------------------------------------------------------------------- inputs
def _limits(case, rng):
    """The rows' limits as 32-bit arrays, None for one that no row has."""
    n, out = case["n"], {}
    for key, dtype, off in (("temperature", np.float32, 1.0), ("top_k", np.int32, 0), ("top_p", np.float32, 1.0), ("min_p", np.float32, 0.0)):
        value = case[key]
        if key != "temperature" and not value:
            out[key] = None
            continue
        a = np.full(n, value, dtype)
        if case["mixed"]:
            spread = np.exp(rng.uniform(-0.5, 0.5, n))
            if key == "top_k":
                a = np.maximum(1, a * spread * spread).astype(dtype)
            elif key == "top_p":
                a = (1.0 - (1.0 - a) * spread).astype(dtype)
            else:
                a = (a * spread).astype(dtype)
            a[rng.random(n) < 0.25] = off
            if key == "temperature":
                a[rng.random(n) < 0.125] = 0.0  # greedy
        out[key] = a
    return out


def _lengths(case, rng):
    """Tokens that each request has in the cache before and after the step."""
    n, longest = case["n"], case["longest"]
    old = np.exp(rng.uniform(0.0, math.log(longest), n)).astype(np.int64)
    kind = case["kind"]
    if kind == "replace":  # of half the requests, some end, some begin, some are cut back to a common beginning
        new = np.exp(rng.uniform(0.0, math.log(longest), n)).astype(np.int64)
        stays = rng.random(n) < 0.5
        new = np.where(stays, np.minimum(old + 1, longest), new)
        new[~stays & (rng.random(n) < 0.25)] = 0
        old[~stays & (rng.random(n) < 0.25)] = 0
    elif kind == "step":
        new = np.minimum(old + 1, longest)
        u = rng.random(n)
        new[u < 1 / 16] = 0                     # ends
        if case["op"] == "tables":
            old[u > 15 / 16] = 0                # begins with its prompt
    else:
        # the step's tokens shared out; in a mixed step most requests have one token, the others a piece of their prompt
        share = rng.exponential(1.0, n)
        running = rng.random(n) < (0.75 if kind == "mixed" else 0.0)
        share[running] = 0
        room = max(0, int(case["tokens"] * 0.95) - int(running.sum()))
        more = np.floor(share / max(share.sum(), 1e-9) * room).astype(np.int64)
        more[running] = 1
        more = np.minimum(more, longest)
        old = np.minimum(old, longest - more)
        if kind == "prompts":                   # some of them share a beginning that is in the cache already
            old[rng.random(n) < 0.75] = 0
        new = old + more
    return old, new


def prepare(case, seed):
    rng = np.random.default_rng(int(seed))
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    n = case["n"]
    s = {"case": case}
    if case["op"] == "sample":
        vocab = case["vocab"]
        x = torch.randn(n, case["pitch"], generator=g, device="cuda").mul_(2.5)
        head = torch.exp(torch.rand(n, HEAD, generator=g, device="cuda", dtype=torch.float64) * math.log(vocab + 1.0)) - 1.0
        lead = 4 + 16 * torch.rand(n, 1, generator=g, device="cuda")
        x.scatter_add_(1, head.long().clamp_(0, vocab - 1), lead / (1 + 0.15 * torch.arange(HEAD, device="cuda")))
        if case["masked"]:  # every second id from a third of the vocabulary on is not allowed
            x[:, vocab // 3:vocab:2] = -math.inf
        s["logits"] = x.to(TYPES[case["type"]])[:, :vocab]
        u = rng.random(n)
        if case["padded"]:  # one row in eight has no request
            u[rng.random(n) < 0.125] = -1.0
        s["uniform"] = torch.from_numpy(u).cuda()
        for key, a in _limits(case, rng).items():
            s[key] = None if a is None else torch.from_numpy(a).cuda()
    else:
        old, new = _lengths(case, rng)
        block = case["block"]
        columns = s["columns"] = -(-case["longest"] // block)
        if case["op"] == "tables":  # the pool holds a third of what all requests could ask for; those that do not fit wait outside
            size = n * columns // 3 + 4 * columns
            waits = np.cumsum(np.maximum(-(-old // block), -(-new // block))) > size
            old[waits] = new[waits] = 0
        held = -(-(old if case["op"] == "tables" else new) // block)
        used = int(held.sum())
        tables = np.full((n, columns), -1, np.int32)
        if case["op"] == "tables":
            blocks = rng.permutation(size).astype(np.int32)
            s["queue"] = torch.from_numpy(np.roll(np.concatenate([blocks[used:], np.full(used, -1, np.int32)]), 5 * int(seed))).cuda()
            head = 5 * int(seed) % size + size * int(rng.integers(1, 1000))
            s["state"] = torch.tensor([head, head + size - used, 0], dtype=torch.int64, device="cuda")
            s["state_out"] = torch.zeros(3, dtype=torch.int64, device="cuda")
        else:
            blocks = rng.permutation(used + 64).astype(np.int32)
        tables[np.arange(columns)[None, :] < held[:, None]] = blocks[:used]
        flat = torch.empty(n * columns + 1, dtype=torch.int32, device="cuda")  # the last element: what no request asks for
        flat[:-1] = torch.from_numpy(tables.ravel()).cuda()
        s["flat"], s["tables"] = flat, flat[:-1].view(n, columns)
        s["old"], s["new"] = (torch.from_numpy(a.astype(np.int32)).cuda() for a in (old, new))
    if own:
        s["tok"] = _tokenizer()
        if case["op"] == "sample":
            s["ids"] = torch.empty(n, device="cuda", dtype=torch.int32)
            s["logprob"] = torch.empty(n, device="cuda")
        elif case["op"] == "slots":
            s["slots"] = torch.empty(case["tokens"], device="cuda", dtype=torch.int64)
            s["positions"], s["requests"] = (torch.empty(case["tokens"], device="cuda", dtype=torch.int32) for _ in range(2))
            s["offsets"] = torch.empty(n + 1, device="cuda", dtype=torch.int64)
    return s


# ---------------------------------------------------------------------------------------------------- the calls
def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _run_own(s):
    case, tok = s["case"], s["tok"]
    if case["op"] == "sample":
        tok.sample(s["logits"].data_ptr(), case["type"], case["n"], case["vocab"], s["uniform"].data_ptr(), s["ids"].data_ptr(),
                   d_logprob=s["logprob"].data_ptr(), d_temperature=_ptr(s["temperature"]), d_top_k=_ptr(s["top_k"]), d_top_p=_ptr(s["top_p"]),
                   d_min_p=_ptr(s["min_p"]), stride=case["pitch"])
        return [s["ids"], s["logprob"]]
    if case["op"] == "tables":
        tok.block_tables(s["old"].data_ptr(), s["new"].data_ptr(), case["n"], case["block"], s["tables"].data_ptr(), s["columns"],
                         s["queue"].data_ptr(), s["queue"].numel(), s["state"].data_ptr(), s["state_out"].data_ptr())
        return [s["tables"], s["queue"], s["state_out"]]
    tok.slot_map(s["old"].data_ptr(), s["new"].data_ptr(), case["n"], case["block"], s["tables"].data_ptr(), s["columns"], case["tokens"],
                 s["slots"].data_ptr(), s["offsets"].data_ptr(), d_positions=s["positions"].data_ptr(), d_requests=s["requests"].data_ptr())
    return [s["slots"], s["positions"], s["requests"], s["offsets"]]


# ---------------------------------------------------------------------------------------------------- the plain forms
def _run_sample(s):
    x, u = s["logits"].float(), s["uniform"]
    n, vocab = x.shape
    t, top_k, top_p, min_p = s["temperature"], s["top_k"], s["top_p"], s["min_p"]
    greedy = t == 0
    high = x.amax(1, keepdim=True)
    y = (x.double() - high.double()) / torch.where(greedy, torch.ones_like(t), t).double()[:, None]
    if top_k is None and top_p is None and min_p is None:
        w = y.exp()
    else:
        best, order = torch.sort(x, dim=1, descending=True, stable=True)
        ys = y.gather(1, order)
        ws = ys.exp()
        place = torch.arange(vocab, device="cuda")[None, :]
        kept = best > -math.inf
        if top_k is not None:
            kept &= (place < top_k[:, None]) | (top_k[:, None] <= 0)
        ws = torch.where(kept, ws, torch.zeros_like(ws))
        if top_p is not None:
            upto = ws.cumsum(1)
            kept &= (upto - ws < top_p.double()[:, None] * upto[:, -1:]) | (top_p[:, None] >= 1)
        if min_p is not None:
            kept &= ys >= min_p.double().log()[:, None]
        kept[:, 0] = True
        w = torch.zeros_like(ws).scatter_(1, order, torch.where(kept, ws, torch.zeros_like(ws)))
    first = torch.where(x == high, torch.arange(vocab, device="cuda")[None, :], vocab).amin(1)
    upto = w.cumsum(1)
    total = upto[:, -1]
    ids = torch.searchsorted(upto, (u * total)[:, None], right=True)[:, 0]
    ids = torch.where(greedy, first, ids.clamp(max=vocab - 1))
    logprob = y.gather(1, ids[:, None])[:, 0] - total.log()
    logprob = torch.where(greedy, torch.zeros_like(logprob), logprob)
    there = u >= 0
    ids = torch.where(there, ids, torch.full_like(ids, -1))
    return [ids.to(torch.int32), torch.where(there, logprob, torch.zeros_like(logprob)).float()]


def _run_tables(s):
    case, columns, queue = s["case"], s["columns"], s["queue"]
    block, size = case["block"], queue.numel()
    old, new = s["old"].long(), s["new"].long()
    there = (old >= 0) & (new >= 0)
    have, need = (old + block - 1) // block, (new + block - 1) // block
    grow = torch.where(there, (need - have).clamp(min=0), 0)
    back = torch.where(there, (have - need).clamp(min=0), 0)
    grown, given = grow.cumsum(0), back.cumsum(0)
    head, tail = s["state"][0], s["state"][1]
    missing = (grown[-1] - (tail - head)).clamp(min=0)
    fits = missing == 0
    i = torch.arange(size, device="cuda")
    # the i-th block that is taken
    r = torch.searchsorted(grown, i, right=True).clamp(max=case["n"] - 1)
    at = r * columns + have[r] + i - (grown - grow)[r]
    taken = (i < grown[-1]) & fits
    # the i-th that is given back
    q = torch.searchsorted(given, i, right=True).clamp(max=case["n"] - 1)
    from_ = q * columns + need[q] + i - (given - back)[q]
    returned = (i < given[-1]) & fits
    to = (tail + i) % size
    flat, none = s["flat"], torch.full_like(i, s["flat"].numel() - 1)
    blocks = flat[torch.where(returned, from_, none)]
    flat.index_put_((torch.where(taken, at, none),), queue[(head + i) % size])
    queue.index_put_((to,), torch.where(returned, blocks, queue[to]))
    zero = torch.zeros_like(missing)
    s["state_out"].copy_(torch.stack([head + torch.where(fits, grown[-1], zero), tail + torch.where(fits, given[-1], zero), missing]))
    return [s["tables"], queue, s["state_out"]]


def _run_slots(s):
    case, block = s["case"], s["case"]["block"]
    old, new = s["old"].long(), s["new"].long()
    more = torch.where((old >= 0) & (new >= 0), (new - old).clamp(min=0), 0)
    upto = more.cumsum(0)
    offsets = torch.cat([torch.zeros_like(upto[:1]), upto])
    i = torch.arange(case["tokens"], device="cuda")
    r = torch.searchsorted(upto, i, right=True).clamp(max=case["n"] - 1)
    there = i < upto[-1]
    position = torch.where(there, old[r] + i - offsets[r], torch.zeros_like(i))
    slots = s["flat"][r * s["columns"] + position // block].long() * block + position % block
    none = torch.full_like(i, -1)
    return [torch.where(there, slots, none), torch.where(there, position, none).to(torch.int32), torch.where(there, r, none).to(torch.int32),
            offsets]


def run(s):
    if own:
        return _run_own(s)
    return {"sample": _run_sample, "tables": _run_tables, "slots": _run_slots}[s["case"]["op"]](s)


# ---------------------------------------------------------------------------------------------------- the definitions
def _exact_sample(s):
    """Rows in blocks; logits as whole numbers in their order with the column behind them, so that no two are alike."""
    case = s["case"]
    n, vocab = case["n"], case["vocab"]
    column = torch.arange(vocab, device="cuda")
    ids, logprobs = [], []
    step = max(1, (1 << 25) // vocab)
    for a in range(0, n, step):
        b = min(n, a + step)
        x = s["logits"][a:b].to(torch.float64)
        t = s["temperature"][a:b].to(torch.float64)
        bits = s["logits"][a:b].float().contiguous().view(torch.int32).long()
        key = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF)) * (1 << 20) + (vocab - 1 - column)[None, :]
        key, order = key.sort(dim=1)
        key, order = key.flip(1), order.flip(1)
        x = x.gather(1, order)
        allowed = ~torch.isneginf(x)
        z = torch.where(allowed, (x - x[:, :1]) / torch.where(t > 0, t, 1.0)[:, None], -math.inf)
        count = allowed.sum(1)
        if s["top_k"] is not None:
            k = s["top_k"][a:b].long()
            count = torch.where(k > 0, torch.minimum(count, k), count)
        upto = torch.where(column[None, :] < count[:, None], z.exp(), 0.0).cumsum(1)
        if s["top_p"] is not None:
            p = s["top_p"][a:b].to(torch.float64)
            reached = 1 + torch.searchsorted(upto, (p * upto[:, -1])[:, None], right=False)[:, 0]
            count = torch.where(p < 1, torch.minimum(count, reached), count)
        if s["min_p"] is not None:
            count = torch.minimum(count, (z >= torch.log(s["min_p"][a:b].to(torch.float64))[:, None]).sum(1))
        count = torch.where(t > 0, count, 1).clamp(min=1)
        mass = upto.gather(1, (count - 1)[:, None])[:, 0]
        by_column = order.argsort(1)            # the place of every column
        w = torch.where(by_column < count[:, None], z.exp().gather(1, by_column), 0.0).cumsum(1)
        u = s["uniform"][a:b]
        drawn = (w <= (u * w[:, -1])[:, None]).sum(1)
        lp = z.gather(1, by_column.gather(1, drawn[:, None].clamp(max=vocab - 1)))[:, 0] - mass.log()
        ids.append(torch.where(u >= 0, drawn, -1).to(torch.int32))
        logprobs.append(torch.where((u >= 0) & (t > 0), lp, 0.0))
    return [torch.cat(ids), torch.cat(logprobs)]


def _exact_tables(s):
    case, block = s["case"], s["case"]["block"]
    old, new = (s[k].cpu().numpy().astype(np.int64) for k in ("old", "new"))
    tables, queue = s["tables"].cpu().numpy().copy(), s["queue"].cpu().numpy().copy()
    head, tail, _ = s["state"].tolist()
    start, size = head, len(queue)
    took = gave = 0
    for r in range(case["n"]):
        have, need = -(-old[r] // block), -(-new[r] // block)
        if need > have:
            tables[r, have:need] = queue[(start + took + np.arange(need - have)) % size]
            took += need - have
        elif have > need:
            queue[(tail + gave + np.arange(have - need)) % size] = tables[r, need:have]
            gave += have - need
    return [tables, queue, np.array([head + took, tail + gave, 0], np.int64)]


def _exact_slots(s):
    case, block = s["case"], s["case"]["block"]
    old, new = (s[k].cpu().numpy().astype(np.int64) for k in ("old", "new"))
    tables = s["tables"].cpu().numpy().astype(np.int64)
    slots = np.full(case["tokens"], -1, np.int64)
    positions, requests = (np.full(case["tokens"], -1, np.int32) for _ in range(2))
    offsets = np.zeros(case["n"] + 1, np.int64)
    for r in range(case["n"]):
        at = offsets[r]
        j = np.arange(old[r], new[r])
        slots[at:at + len(j)] = tables[r, j // block] * block + j % block
        positions[at:at + len(j)] = j
        requests[at:at + len(j)] = r
        offsets[r + 1] = at + len(j)
    return [slots, positions, requests, offsets]


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"sample": _exact_sample, "tables": _exact_tables, "slots": _exact_slots}[case["op"]](s)


@functools.lru_cache(maxsize=64)
def _moved(n, block, longest, kind):
    """Blocks that a step takes and gives back, on average."""
    case = {"op": "tables", "n": n, "block": block, "longest": longest, "kind": kind}
    took = gave = 0
    for seed in range(4):
        old, new = _lengths(case, np.random.default_rng(seed))
        d = -(-new // block) + old // -block
        took, gave = took + int(d[d > 0].sum()), gave - int(d[d < 0].sum())
    return took / 4, gave / 4


def work(case):
    n = case["n"]
    if case["op"] == "sample":
        rows = n * 0.875 if case["padded"] else n
        limits = 4 * sum(1 for k in ("top_k", "top_p", "min_p") if case[k])
        return {"bytes": rows * case["vocab"] * SIZE[case["type"]] + n * (8 + 4 + limits + 8), "flops": 4 * rows * case["vocab"]}
    if case["op"] == "tables":
        took, gave = _moved(n, case["block"], case["longest"], case["kind"])
        return {"bytes": 8 * n + 8 * (took + gave) + 48, "flops": 8 * n + took + gave}
    return {"bytes": 8 * n + 4 * (n + case["tokens"] // case["block"]) + 16 * case["tokens"] + 8 * (n + 1), "flops": 4 * case["tokens"]}
