"""The operators at a model's two ends, where token ids go in and come out, as cases that can be timed and compared.

``op`` says which entry point of ``gputok_b200.Tokenizer`` a case goes through:

  embed     embed                 ids to scaled rows of a table
  embed'    embed_grad            the table's gradient
  score     token_logprobs        log probability of given ids, entropy, log-sum-exp and the top alternatives
  score'    token_logprobs_grad   the logits' gradient

With ``own`` false ``run`` computes them in elementary torch operations instead, in 32 bits, rounded once at the end.
Ids are drawn so that id v has a probability of about 1 / v, as in text under a table whose ids are in the order of the
merges; logits are normal with the given id raised, which is what a trained model's look like.
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


def _embed(op, n, vocab, dim, table, rows, scale=1.0, padded=False):
    return {"op": op, "n": n, "vocab": vocab, "dim": dim, "table": table, "rows": rows, "scale": scale, "padded": padded}


def _score(op, n, vocab, type_, top=0, entropy=False, scale=1.0, pitch=0, masked=False, padded=False):
    return {"op": op, "n": n, "vocab": vocab, "type": type_, "top": top, "entropy": entropy, "scale": scale,
            "pitch": pitch or vocab, "masked": masked, "padded": padded}


def listed():
    return [
        # the newest token of one running text
        dict(_embed("embed", 1, GPT2, 768, "bf16", "bf16"), name="embed one token"),
        # 32 texts of 1024 tokens in front of the first layer, scaled by the root of the width
        dict(_embed("embed", 32768, GPT2, 1024, "bf16", "bf16", 32.0), name="embed a batch"),
        # 32-bit weights, 16-bit activations, a width that no vector load divides, texts padded with -1
        dict(_embed("embed", 10007, 32003, 777, "f32", "f16", 1.0, True), name="embed odd rows"),
        # a small model's step: few tokens, a table of a few thousand ids
        dict(_embed("embed'", 512, 8193, 512, "f32", "f32"), name="embed grad, few tokens"),
        # one training step of 32 texts of 1024 tokens, gradient kept in 32 bits
        dict(_embed("embed'", 32768, GPT2, 768, "f32", "bf16"), name="embed grad, a batch"),
        # a long step of a wide model with 16-bit gradients, odd width, padded texts
        dict(_embed("embed'", 131072, GPT2, 1601, "bf16", "bf16", 40.0, True), name="embed grad, long and odd"),
        # one sampled token and its alternatives, as served
        dict(_score("score", 1, GPT2, "bf16", 20, True), name="score one token"),
        # a prompt's tokens with their alternatives; part of the ids is masked; rows padded to a multiple of 64
        dict(_score("score", 999, GPT2, "f32", 5, True, 0.7, 50304, True), name="score a prompt"),
        # the loss of a training step of 8 texts of 1024 tokens
        dict(_score("score", 8192, GPT2, "bf16"), name="score a batch"),
        # the loss's gradient of a few tokens
        dict(_score("score'", 32, GPT2, "bf16", pitch=50304), name="score grad, few tokens"),
        # the loss's gradient of the training step above
        dict(_score("score'", 8192, GPT2, "bf16"), name="score grad, a batch"),
        # policy gradient with an entropy term, odd sizes, masked ids, padded texts
        dict(_score("score'", 1021, 32003, "f16", 0, True, 0.8, 0, True, True), name="score grad with entropy"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "embed'", "score", "score'"])
    vocab = GPT2 if rng.random() < 0.3 else _log(rng, 257, 131072)
    if op[0] == "e":
        dim = min(_log(rng, 33, 4096), (1 << 27) // vocab)
        if rng.random() < 0.6:
            dim = (dim + 7) // 8 * 8
        n = _log(rng, 1, min(131072, (131072 * 1601) // (2 * dim)))
        table = rng.choice(sorted(TYPES))
        rows = table if rng.random() < 0.6 else rng.choice(sorted(TYPES))
        return _embed(op, n, vocab, dim, table, rows, rng.choice([1.0, round(math.sqrt(dim), 3)]), rng.random() < 0.3)
    n = _log(rng, 1, min(8192, (8192 * GPT2) // (2 * vocab)))
    pitch = (vocab + 63) // 64 * 64 if rng.random() < 0.5 else vocab
    top = rng.choice([0, 0, 1, 5, 20, 32]) if op == "score" and n * vocab < 1 << 27 else 0
    return _score(op, n, vocab, rng.choice(sorted(TYPES)), top, rng.random() < 0.5, rng.choice([1.0, 1.0, 0.7, 1.25]), pitch,
                  rng.random() < 0.3, rng.random() < 0.3)


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


def _ids(g, n, vocab, padded):
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    ids = (torch.exp(u * math.log(vocab + 1.0)) - 1.0).long().clamp_(0, vocab - 1).to(torch.int32)
    if padded:  # one id in eight is padding
        ids = torch.where(torch.rand(n, generator=g, device="cuda") < 0.125, torch.full_like(ids, -1), ids)
    return ids


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    n, vocab = case["n"], case["vocab"]
    s = {"case": case, "ids": _ids(g, n, vocab, case["padded"])}
    if case["op"] == "embed":
        s["table"] = (torch.randn(vocab, case["dim"], generator=g, device="cuda") * 0.02).to(TYPES[case["table"]])
    elif case["op"] == "embed'":
        s["grad"] = torch.randn(n, case["dim"], generator=g, device="cuda").to(TYPES[case["rows"]])
    else:
        x = torch.randn(n, case["pitch"], generator=g, device="cuda").mul_(2.5)
        at = s["ids"].clamp(min=0).long()[:, None]
        x.scatter_add_(1, at, torch.rand(n, 1, generator=g, device="cuda") * 12)
        if case["masked"]:  # every second id from a third of the table on is not allowed
            x[:, vocab // 3:vocab:2] = -math.inf
        s["logits"] = x.to(TYPES[case["type"]])[:, :vocab]
        if case["op"] == "score'":
            s["grad_logprob"] = torch.randn(n, generator=g, device="cuda") * 0.1 - 1.0
            s["grad_entropy"] = torch.randn(n, generator=g, device="cuda") * 0.1 if case["entropy"] else None
            z = torch.log_softmax(s["logits"].float() * case["scale"], 1)
            s["entropy"] = -torch.where(z > -math.inf, z.exp() * z, torch.zeros_like(z)).sum(1)
            s["lse"] = torch.logsumexp(s["logits"].float() * case["scale"], 1)
    if own:
        _prepare_own(s)
    return s


def _prepare_own(s):
    case, dev = s["case"], "cuda"
    tok = s["tok"] = _tokenizer()
    n, vocab = case["n"], case["vocab"]
    if case["op"] == "embed":
        s["out"] = torch.empty(n, case["dim"], device=dev, dtype=TYPES[case["rows"]])
    elif case["op"] == "embed'":
        s["out"] = torch.empty(vocab, case["dim"], device=dev, dtype=TYPES[case["table"]])
        s["work"] = torch.empty(tok.embed_grad_workspace(n, vocab, case["dim"]), device=dev, dtype=torch.uint8)
    elif case["op"] == "score":
        k = case["top"]
        s["logprob"] = torch.empty(n, device=dev)
        s["lse"] = torch.empty(n, device=dev)
        s["entropy"] = torch.empty(n, device=dev) if case["entropy"] else None
        s["top_ids"] = torch.empty(n, k, device=dev, dtype=torch.int32) if k else None
        s["top_logprobs"] = torch.empty(n, k, device=dev) if k else None
    else:
        s["out"] = torch.empty(n, case["pitch"], device=dev, dtype=TYPES[case["type"]])[:, :vocab]


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _run_own(s):
    case, tok = s["case"], s["tok"]
    n, vocab = case["n"], case["vocab"]
    if case["op"] == "embed":
        tok.embed(s["ids"].data_ptr(), n, s["table"].data_ptr(), case["table"], vocab, case["dim"], s["out"].data_ptr(), case["rows"],
                  scale=case["scale"])
        return s["out"]
    if case["op"] == "embed'":
        tok.embed_grad(s["ids"].data_ptr(), n, s["grad"].data_ptr(), case["rows"], vocab, case["dim"], s["out"].data_ptr(), case["table"],
                       s["work"].data_ptr(), s["work"].numel(), scale=case["scale"])
        return s["out"]
    if case["op"] == "score":
        tok.token_logprobs(s["logits"].data_ptr(), case["type"], n, vocab, s["ids"].data_ptr(), s["logprob"].data_ptr(),
                           d_entropy=_ptr(s["entropy"]), d_lse=s["lse"].data_ptr(), top_k=case["top"], d_top_ids=_ptr(s["top_ids"]),
                           d_top_logprobs=_ptr(s["top_logprobs"]), scale=case["scale"], stride=case["pitch"])
        return [s["logprob"], s["lse"]] + [t for t in (s["entropy"], s["top_ids"], s["top_logprobs"]) if t is not None]
    tok.token_logprobs_grad(s["logits"].data_ptr(), case["type"], n, vocab, s["ids"].data_ptr(), s["lse"].data_ptr(),
                            s["grad_logprob"].data_ptr(), s["out"].data_ptr(), d_entropy=_ptr(s["entropy"]),
                            d_grad_entropy=_ptr(s["grad_entropy"]), scale=case["scale"], stride=case["pitch"], grad_stride=case["pitch"])
    return s["out"]


def run(s):
    if own:
        return _run_own(s)
    case, ids = s["case"], s["ids"].long()
    kept = ids >= 0
    if case["op"] == "embed":
        rows = s["table"][ids.clamp(min=0)].float() * case["scale"]
        return torch.where(kept[:, None], rows, torch.zeros_like(rows)).to(TYPES[case["rows"]])
    if case["op"] == "embed'":
        out = torch.zeros(case["vocab"], case["dim"], device="cuda")
        rows = torch.where(kept[:, None], s["grad"].float(), torch.zeros((), device="cuda"))
        out.index_add_(0, ids.clamp(min=0), rows)
        return (out * case["scale"]).to(TYPES[case["table"]])
    x = s["logits"].float()
    at = ids.clamp(min=0)[:, None]
    if case["op"] == "score":
        z = (x - x.amax(1, keepdim=True)) * case["scale"]
        log_sum = z.exp().sum(1).log()
        lse = x.amax(1) * case["scale"] + log_sum
        out = [torch.where(kept, z.gather(1, at)[:, 0] - log_sum, torch.zeros_like(log_sum)), lse]
        if case["entropy"]:
            z = z - log_sum[:, None]
            out.append(-torch.where(z > -math.inf, z.exp() * z, torch.zeros_like(z)).sum(1))
        if case["top"]:
            best, which = torch.sort(x, dim=1, descending=True, stable=True)
            best, which = best[:, :case["top"]], which[:, :case["top"]]
            out.append(torch.where(best > -math.inf, which, torch.full_like(which, -1)).to(torch.int32))
            out.append((best - x.amax(1, keepdim=True)) * case["scale"] - log_sum[:, None])
        return out
    z = x * case["scale"] - s["lse"][:, None]
    p = z.exp()
    g = torch.where(kept, s["grad_logprob"], torch.zeros_like(s["grad_logprob"]))
    d = -p * g[:, None]
    d.scatter_add_(1, at, g[:, None])
    if case["entropy"]:
        z = torch.where(z > -math.inf, z, torch.zeros_like(z))
        d = d - s["grad_entropy"][:, None] * p * (z + s["entropy"][:, None])
    d = (d * case["scale"]).to(TYPES[case["type"]])
    out = torch.empty(case["n"], case["pitch"], device="cuda", dtype=d.dtype)[:, :case["vocab"]]
    return out.copy_(d)


def exact(case, seed):
    """The definitions in 64 bits, block of rows by block of rows."""
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    ids = s["ids"].cpu().numpy()
    n, vocab, f64 = case["n"], case["vocab"], torch.float64
    if case["op"] == "embed":
        out = torch.zeros(n, case["dim"], device="cuda", dtype=f64)
        at = torch.from_numpy(np.flatnonzero(ids >= 0)).cuda()
        out[at] = torch.index_select(s["table"], 0, s["ids"][at]).to(f64) * case["scale"]
        return out
    if case["op"] == "embed'":
        # sorted tokens, sums between the places where the id changes
        order = np.argsort(ids, kind="stable")
        order = order[ids[order] >= 0]
        found, first = np.unique(ids[order], return_index=True)
        out = torch.zeros(vocab, case["dim"], device="cuda", dtype=f64)
        order_d = torch.from_numpy(order).cuda()
        counts = torch.from_numpy(np.diff(np.append(first, len(order)))).cuda()
        step = max(1, (1 << 27) // n)
        for c in range(0, case["dim"] if len(order) else 0, step):
            part = s["grad"][:, c:c + step].to(f64)[order_d]
            out[torch.from_numpy(found).long().cuda(), c:c + step] = torch.segment_reduce(part, "sum", lengths=counts, axis=0)
        return out * case["scale"]
    k, parts = case["top"], []
    step = max(1, (1 << 26) // vocab)
    row = torch.arange(vocab, device="cuda")
    for a in range(0, n, step):
        b = min(n, a + step)
        raw = s["logits"][a:b].to(f64)
        t = s["ids"][a:b].long()
        here = row[None, :] == t[:, None]
        z = raw * case["scale"]
        allowed = torch.isfinite(z)
        if case["op"] == "score":
            lse = torch.logsumexp(z, 1)
            logp = z - lse[:, None]
            lp = torch.where(here, logp, torch.zeros_like(logp)).sum(1)
            got = [lp, lse]
            if case["entropy"]:
                got.append(torch.where(allowed, -logp.exp() * logp, torch.zeros_like(logp)).sum(1))
            if k:
                # logits as whole numbers in their order, the column behind them: no two alike
                bits = s["logits"][a:b].float().contiguous().view(torch.int32).long()
                key = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF)) * (1 << 20) + (vocab - 1 - row)[None, :]
                key, which = torch.topk(key, k, dim=1)
                fine = allowed.gather(1, which)
                got.append(torch.where(fine, which, torch.full_like(which, -1)).to(torch.int32))
                got.append(logp.gather(1, which))
            parts.append(got)
            continue
        logp = z - torch.logsumexp(z, 1, keepdim=True)
        p = logp.exp()
        g = torch.where(t >= 0, s["grad_logprob"][a:b], torch.zeros_like(s["grad_logprob"][a:b])).to(f64)[:, None]
        d = g * (here.to(f64) - p)
        if case["entropy"]:
            inner = torch.where(allowed, p * logp, torch.zeros_like(p))
            d = d - s["grad_entropy"][a:b].to(f64)[:, None] * (inner - p * inner.sum(1, keepdim=True))
        parts.append([d * case["scale"]])
    out = [torch.cat(p) for p in zip(*parts)]
    return out if case["op"] == "score" else out[0]


@functools.lru_cache(maxsize=64)
def _distinct(n, vocab):
    """How many different ids n draws are expected to hold."""
    edges = np.log1p(np.arange(vocab + 1, dtype=np.float64)) / math.log(vocab + 1.0)
    return float(-np.expm1(n * np.log1p(-np.minimum(np.diff(edges), 1 - 1e-12))).sum())


def work(case):
    n, vocab = case["n"], case["vocab"]
    if case["op"][0] == "e":
        kept = n * 0.875 if case["padded"] else n
        dim, rows, table = case["dim"], SIZE[case["rows"]], SIZE[case["table"]]
        if case["op"] == "embed":
            return {"bytes": 4 * n + _distinct(int(kept) or 1, vocab) * dim * table + n * dim * rows, "flops": kept * dim}
        return {"bytes": 4 * n + kept * dim * rows + vocab * dim * table, "flops": kept * dim}
    size = SIZE[case["type"]]
    if case["op"] == "score":
        return {"bytes": n * vocab * size + n * (12 + (4 if case["entropy"] else 0) + 8 * case["top"]),
                "flops": n * vocab * (6 if case["entropy"] else 4)}
    return {"bytes": 2 * n * vocab * size + n * (12 + (8 if case["entropy"] else 0)), "flops": n * vocab * (8 if case["entropy"] else 4)}
