"""The operators at a model's two ends (ids to rows of a table, logits to log probabilities, and their gradients)
against plain implementations in 64 bits, through the C ABI.

Tolerances are bounds, not measurements: u = 2^-24 is half a step of a 32-bit float, a sum of n numbers in any order is
off by at most (n - 1) u times the sum of their sizes, and storing a value costs half a step of its type.
"""
from __future__ import annotations

import math

import numpy as np
import pytest

from gputok_b200 import GtkError, Tokenizer, load_library

U = 2.0 ** -24
TYPES = ("f32", "bf16", "f16")


# ---------------------------------------------------------------------------------------------------- refusals (CPU)
@pytest.fixture(scope="module")
def host(native_built, merges_path):
    return Tokenizer(merges_path, 2048, 50, device=-1)


P = 1 << 20  # an address that no refused call gets to use

EMBED = dict(d_ids=P, n_ids=3, d_table=P, table_type="f32", vocab=10, dim=8, d_out=P, out_type="f32")
EMBED_GRAD = dict(d_ids=P, n_ids=3, d_grad_out=P, out_type="f32", vocab=10, dim=8, d_grad_table=P, table_type="f32", d_workspace=P,
                  workspace_bytes=1 << 30)
SCORE = dict(d_logits=P, type="f32", n_rows=3, vocab=10, d_targets=P, d_logprob=P, d_entropy=P, d_lse=P, top_k=5, d_top_ids=P,
             d_top_logprobs=P)
SCORE_GRAD = dict(d_logits=P, type="f32", n_rows=3, vocab=10, d_targets=P, d_lse=P, d_grad_logprob=P, d_grad_logits=P, d_entropy=P,
                  d_grad_entropy=P)

REFUSED = [
    ("embed", EMBED, [dict(n_ids=-1), dict(vocab=0), dict(dim=0), dict(n_ids=1 << 31), dict(vocab=1 << 31), dict(dim=(1 << 20) + 1),
                      dict(table_stride=-1), dict(out_stride=7), dict(d_ids=0), dict(d_table=0), dict(d_out=0), dict(d_ids=P + 2),
                      dict(d_table=P + 2), dict(d_out=P + 2), dict(d_out=P + 1, out_type="bf16")]),
    ("embed_grad", EMBED_GRAD, [dict(n_ids=-1), dict(vocab=0), dict(dim=0), dict(n_ids=1 << 31), dict(vocab=1 << 31), dict(dim=(1 << 20) + 1),
                                dict(out_stride=-1), dict(table_stride=7), dict(d_ids=0), dict(d_grad_out=0), dict(d_grad_table=0),
                                dict(d_workspace=0), dict(d_workspace=P + 8), dict(workspace_bytes=255), dict(d_ids=P + 1),
                                dict(d_grad_out=P + 2), dict(d_grad_table=P + 1, table_type="f16"), dict(n_ids=0, d_grad_table=0)]),
    ("token_logprobs", SCORE, [dict(n_rows=-1), dict(vocab=0), dict(n_rows=1 << 31), dict(vocab=(1 << 30) + 1), dict(stride=-1),
                               dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan), dict(top_k=-1),
                               dict(top_k=33), dict(top_k=0), dict(d_top_ids=0, d_top_logprobs=0), dict(d_logits=0), dict(d_targets=0),
                               dict(d_logits=P + 2), dict(d_logits=P + 1, type="bf16"), dict(d_targets=P + 2), dict(d_lse=P + 1),
                               dict(d_top_ids=P + 2)]),
    ("token_logprobs_grad", SCORE_GRAD, [dict(n_rows=-1), dict(vocab=0), dict(n_rows=1 << 31), dict(vocab=(1 << 30) + 1), dict(stride=-1),
                                         dict(grad_stride=9), dict(scale=0.0), dict(scale=math.nan), dict(d_logits=0), dict(d_lse=0),
                                         dict(d_targets=0), dict(d_grad_logits=0), dict(d_entropy=0), dict(d_grad_logits=P + 2),
                                         dict(d_logits=P + 1, type="f16"), dict(d_lse=P + 2), dict(stride=16, grad_stride=10)]),
]


@pytest.mark.parametrize("name,good,change", [(n, g, c) for n, g, cs in REFUSED for c in cs],
                         ids=lambda v: v if isinstance(v, str) else ",".join(f"{k}={x}" for k, x in v.items()) if len(v) < 3 else "")
def test_refused_arguments(host, name, good, change):
    with pytest.raises(GtkError) as e:
        getattr(host, name)(**{**good, **change})
    assert e.value.code == 1 and len(str(e.value)) > 30


@pytest.mark.parametrize("name,good", [(n, g) for n, g, _ in REFUSED])
def test_host_only_handle_has_no_operators(host, name, good):
    with pytest.raises(GtkError) as e:
        getattr(host, name)(**good)
    assert e.value.code == 6


def test_unknown_types_and_null_handles(host):
    lib = load_library()
    assert lib.gtk_embed(host._h, P, 1, P, 3, 10, 8, 8, 1.0, P, 0, 8) == 1
    assert lib.gtk_embed(host._h, P, 1, P, 0, 10, 8, 8, 1.0, P, -1, 8) == 1
    assert lib.gtk_token_logprobs(host._h, P, 7, 1, 10, 10, 1.0, P, 0, P, None, None, None, None) == 1
    assert lib.gtk_embed(None, P, 1, P, 0, 10, 8, 8, 1.0, P, 0, 8) == 1
    assert lib.gtk_embed_grad_workspace(None, 1, 1, 1, None) == 1
    assert lib.gtk_embed_grad_workspace(host._h, 1, 1, 1, None) == 1
    with pytest.raises(GtkError):
        host.embed_grad_workspace(1, 0, 1)


def test_workspace_sizes(host):
    """Enough for what the call keeps: sorted ids, and parts of sums; never beyond a small multiple of it."""
    for n in (0, 1, 7, 4096, 131072, 1 << 22):
        for vocab in (1, 257, 50257, 131072):
            for dim in (1, 64, 777, 4096):
                need = host.embed_grad_workspace(n, vocab, dim)
                assert need >= 8 * n and need % 256 == 0
                assert need < 64 * n + 4 * vocab + 48 * (1 << 20) + 64 * 8 * dim


LONG_SUMS = r"""
#include "gtk_long_sums.hpp"
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

// Owners of ids by id % 8 on tokens grouped by owner, then id, those of no id last: every place that is asked about and every block
// that is put, from all owners' threads.
int main()
{
  std::mt19937 rng(7);
  long outside = 0, twice = 0, missing = 0, wrong = 0, owners_without = 0;
  for (int round = 0; round < 20000; ++round) {
    const int log2 = 1 + int(rng() % 3), vocab = 1 + int(rng() % 40), none = int(rng() % 3 ? 0 : rng() % 9);
    const int64_t kept = rng() % 90, n = kept + none;
    const int kinds = 1 + int(rng() % vocab);
    std::vector<uint32_t> ids(n, 0xFFFFFFFFu);
    for (int64_t i = 0; i < kept; ++i) ids[i] = rng() % kinds;
    std::sort(ids.begin(), ids.begin() + kept, [](uint32_t a, uint32_t b) { return a % 8 != b % 8 ? a % 8 < b % 8 : a < b; });
    const int64_t blocks = (n + (1 << log2) - 1) >> log2;
    std::vector<int> puts(blocks, 0);
    std::vector<gtk::LongSum> got(blocks, gtk::LongSum{0, 99});
    for (int64_t i = kept; i < n; ++i)  // the blocks that end behind the last share
      if (i + 1 == n || (i + 1) % (1 << log2) == 0) ++puts[i >> log2], got[i >> log2] = gtk::LongSum{0xFFFFFFFFu, 0};
    int64_t begin = 0;
    for (uint32_t owner = 0; owner < 8; ++owner) {
      int64_t end = begin;
      while (end < kept && ids[end] % 8 == owner) ++end;
      owners_without += begin == end;
      for (int thread = 0; thread < 4; ++thread)
        gtk::each_long_sum(
            begin, end, n, log2, thread, 4,
            [&](int64_t place) {
              if (place < begin || place >= end) ++outside;
              return place < 0 || place >= n ? 0u : ids[place];
            },
            [&](int64_t block, const gtk::LongSum& L) {
              if (block < 0 || block >= blocks) return void(++outside);
              ++puts[block];
              got[block] = L;
            });
      begin = end;
    }
    std::vector<uint32_t> parts(blocks, 0);
    for (int64_t s = 0; s < kept;) {
      int64_t e = s;
      while (e < kept && ids[e] == ids[s]) ++e;
      const int64_t a = s >> log2, b = (e - 1) >> log2;
      if (b >= a + 2) parts[a] = uint32_t(b - a + 1);
      s = e;
    }
    for (int64_t b = 0; b < blocks; ++b) {
      twice += puts[b] > 1, missing += puts[b] == 0;
      const int64_t last = std::min((b + 1) << log2, n) - 1;
      wrong += puts[b] && (got[b].parts != parts[b] || (parts[b] && got[b].id != ids[last]));
    }
  }
  std::printf("outside=%ld twice=%ld missing=%ld wrong=%ld\n", outside, twice, missing, wrong);
  return owners_without > 1000 ? 0 : 1;
}
"""


def test_long_sums_are_found_by_one_owner_from_its_own_tokens(tmp_path):
    """What k_embed_grad_sort does to find the sums that are cut into parts, run on the CPU: no owner looks at another's tokens, which
    that one may be moving, and each block's entry is one owner's, those without tokens included."""
    import os
    import subprocess

    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gpu-tokenizer_b200", "csrc")
    (tmp_path / "t.cpp").write_text(LONG_SUMS)
    subprocess.run(["g++", "-O1", "-std=c++17", "-I", csrc, "t.cpp", "-o", "t"], cwd=tmp_path, check=True)
    run = subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and run.stdout == "outside=0 twice=0 missing=0 wrong=0\n", run.stdout


# ---------------------------------------------------------------------------------------------------- on the GPU
@pytest.fixture(scope="module")
def tok(native_built, merges_path):
    import torch

    t = Tokenizer(merges_path, 2048, 50, device=0)
    t.set_stream(torch.cuda.current_stream().cuda_stream)
    return t


def dtype(name):
    import torch

    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


def half_step(name):
    import torch

    return torch.finfo(dtype(name)).eps / 2


def tiny(name):
    """Half a step among the subnormals."""
    import torch

    fi = torch.finfo(dtype(name))
    return fi.smallest_normal * fi.eps / 2


def rows(values, name, stride=None, shift=0):
    """The values (n x d) in an array of the type with a stride and a first element `shift` elements behind an aligned one;
    what lies around holds a mark.  Returns (whole array, view)."""
    import torch

    n, d = values.shape
    stride = d if stride is None else stride
    whole = torch.full((n * stride + shift + 16,), 7.5, device="cuda", dtype=dtype(name))
    view = whole[shift:].as_strided((n, d), (stride, 1))
    view.copy_(values)
    return whole, view


def marks_untouched(whole, n, d, stride, shift):
    import torch

    keep = torch.ones_like(whole, dtype=torch.bool)
    keep[shift:].as_strided((n, d), (stride, 1)).fill_(False)
    return bool((whole[keep] == 7.5).all())


def some_ids(seed, n, vocab, kind):
    """int32 ids on the GPU: 'text' (id v about as often as 1 / v), 'one' (all the same), 'all' (every id once, shuffled),
    'padded' (text with negative ids), 'wrong' (some >= vocab too)."""
    import torch

    g = torch.Generator().manual_seed(seed)
    ids = (torch.exp(torch.rand(n, generator=g, dtype=torch.float64) * math.log(vocab + 1.0)) - 1).long().clamp(0, vocab - 1)
    if kind == "one":
        ids[:] = vocab // 2
    if kind == "all":
        ids = torch.randperm(max(n, vocab), generator=g)[:n] % vocab
    if kind in ("padded", "wrong"):
        ids[torch.rand(n, generator=g) < 0.3] = -1
        ids[torch.rand(n, generator=g) < 0.05] = -(1 << 31)
    if kind == "wrong":
        ids[torch.rand(n, generator=g) < 0.1] = vocab
        ids[torch.rand(n, generator=g) < 0.05] = (1 << 31) - 1
    return ids.to(torch.int32).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("table_type", TYPES)
@pytest.mark.parametrize("out_type", TYPES)
@pytest.mark.parametrize("n,vocab,dim,ts,os,shift,kind", [
    (1, 50257, 768, 768, 768, 0, "text"),
    (1, 1, 1, 1, 1, 0, "one"),
    (2, 300, 8, 16, 24, 0, "wrong"),
    (33, 300, 100, 104, 128, 0, "padded"),       # rows aligned, their length no multiple of a pack
    (257, 1000, 777, 777, 780, 1, "wrong"),
    (100, 511, 1024, 1024, 1024, 1, "text"),     # packs would fit, the first element is not aligned
    (65, 90, 4100, 4104, 4100, 0, "text"),
    (4099, 5000, 256, 256, 256, 0, "padded"),
    (50, 40, 64, 0, 64, 0, "text"),              # every row of the table is the same one
])
def test_embed(tok, table_type, out_type, n, vocab, dim, ts, os, shift, kind):
    import torch

    g = torch.Generator(device="cuda").manual_seed(n + dim)
    values = torch.randn(1 if ts == 0 else vocab, dim, generator=g, device="cuda")
    _, table = rows(values, table_type, max(ts, dim), shift)
    out_all, out = rows(torch.zeros(n, dim, device="cuda"), out_type, os, shift)
    ids = some_ids(n, n, vocab, kind)
    scale = 1.7
    tok.embed(ids.data_ptr(), n, table.data_ptr(), table_type, vocab, dim, out.data_ptr(), out_type, scale=scale, table_stride=ts,
              out_stride=os)
    fine = (ids >= 0) & (ids < vocab)
    want = table.double()[torch.zeros_like(ids) if ts == 0 else torch.where(fine, ids, torch.zeros_like(ids))]
    want = want * float(np.float32(scale))
    want = torch.where(fine[:, None], want, torch.zeros_like(want))
    got = out.double()
    assert bool((torch.isnan(got) == (ids >= vocab)[:, None]).all())
    want = torch.where((ids >= vocab)[:, None], got, want)
    # one product in 32 bits, one rounding to the type
    err = (got - want).abs() - (want.abs() * (U + half_step(out_type) * (1 + U)) + tiny(out_type))
    assert not bool((err > 0).any())
    assert marks_untouched(out_all, n, dim, os, shift)


@pytest.mark.gpu
def test_embed_of_nothing(tok):
    import torch

    out = torch.full((8,), 3.0, device="cuda")
    tok.embed(0, 0, 0, "f32", 10, 8, 0, "f32")
    tok.embed(out.data_ptr(), 0, out.data_ptr(), "f32", 10, 8, out.data_ptr(), "f32")
    assert bool((out == 3).all())


def embed_grad(tok, ids, grad, grad_type, vocab, dim, table, table_type, spare=0, **more):
    import torch

    n = ids.numel()
    need = tok.embed_grad_workspace(n, vocab, dim)
    work = torch.full((need + spare,), 0xAB, device="cuda", dtype=torch.uint8)
    tok.embed_grad(ids.data_ptr(), n, grad.data_ptr(), grad_type, vocab, dim, table.data_ptr(), table_type, work.data_ptr(), need, **more)
    return work


def check_embed_grad(ids, grad, vocab, dim, scale, base, got, table_type):
    """Against the formula, with the bound that the number of summands gives."""
    import torch

    fine = (ids >= 0) & (ids < vocab)
    at = ids[fine].long()
    dy = grad.double()[fine]
    scale = float(np.float32(scale))
    total = torch.zeros(vocab, dim, device="cuda", dtype=torch.float64).index_add_(0, at, dy) * scale
    size = torch.zeros(vocab, dim, device="cuda", dtype=torch.float64).index_add_(0, at, dy.abs()) * scale
    count = torch.zeros(vocab, device="cuda", dtype=torch.float64).index_add_(0, at, torch.ones_like(at, dtype=torch.float64))
    want = total if base is None else base.double() + total
    # the sum, the product with scale, the base's addition, the rounding to the type
    bound = size * (count[:, None] + 2) * U * 1.01 + want.abs() * (U + half_step(table_type) * 1.01) + tiny(table_type) + 1e-44
    if base is not None:
        bound = torch.where((count > 0)[:, None], bound, torch.zeros_like(bound))  # rows that no id points to are not touched
    else:
        assert bool((got[count == 0] == 0).all())
    err = (got.double() - want).abs() - bound
    assert not bool((err > 0).any()), float(err.max())


GRAD_CASES = [
    (1, 50257, 768, 768, 768, 0, "text"),
    (1, 1, 1, 1, 1, 0, "one"),
    (7, 300, 8, 16, 24, 0, "wrong"),
    (33, 300, 100, 104, 128, 0, "padded"),
    (600, 300, 100, 100, 100, 0, "one"),        # one sum over many units
    (513, 1000, 777, 777, 780, 1, "wrong"),
    (2048, 4096, 36, 40, 36, 0, "all"),
    (2049, 257, 264, 264, 264, 0, "text"),
    (5000, 70000, 64, 64, 72, 0, "padded"),     # ids beyond 16 bits
    (9000, 600, 333, 333, 333, 0, "text"),
    (40001, 50257, 96, 96, 96, 0, "text"),
    (5000, 40, 64, 0, 64, 0, "text"),           # the same gradient for every token
    (30, 300, 2050, 2056, 2056, 0, "text"),
    (300, 12, 64, 64, 64, 0, "empty"),          # nothing but padding
]


@pytest.mark.gpu
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("grad_type,table_type", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("n,vocab,dim,gs,ts,shift,kind", GRAD_CASES)
def test_embed_grad(tok, grad_type, table_type, n, vocab, dim, gs, ts, shift, kind, accumulate):
    import torch

    g = torch.Generator(device="cuda").manual_seed(n + dim)
    _, grad = rows(torch.randn(1 if gs == 0 else n, dim, generator=g, device="cuda"), grad_type, max(gs, dim), shift)
    ids = some_ids(n, n, vocab, "text" if kind == "empty" else kind)
    if kind == "empty":
        ids.fill_(-1)
    start = torch.randn(vocab, dim, generator=g, device="cuda")
    whole, table = rows(start, table_type, ts, shift)
    base = table.clone() if accumulate else None
    embed_grad(tok, ids, grad, grad_type, vocab, dim, table, table_type, scale=0.75, accumulate=accumulate, out_stride=gs, table_stride=ts)
    check_embed_grad(ids, grad.expand(n, dim) if gs == 0 else grad, vocab, dim, 0.75, base, table, table_type)
    assert marks_untouched(whole, vocab, dim, ts, shift)
    again_whole, again = rows(start, table_type, ts, shift)     # the same ids: the same bits
    embed_grad(tok, ids, grad, grad_type, vocab, dim, again, table_type, scale=0.75, accumulate=accumulate, out_stride=gs, table_stride=ts)
    assert torch.equal(again, table)


def run_embed_grad(tok, grad_type, table_type, n, vocab, dim, gs, ts, shift, kind, accumulate):
    import torch

    g = torch.Generator(device="cuda").manual_seed(n + dim)
    _, grad = rows(torch.randn(1 if gs == 0 else n, dim, generator=g, device="cuda"), grad_type, max(gs, dim), shift)
    ids = some_ids(n, n, vocab, "text" if kind == "empty" else kind)
    if kind == "empty":
        ids.fill_(-1)
    whole, table = rows(torch.randn(vocab, dim, generator=g, device="cuda"), table_type, ts, shift)
    base = table.clone() if accumulate else None
    embed_grad(tok, ids, grad, grad_type, vocab, dim, table, table_type, scale=0.75, accumulate=accumulate, out_stride=gs, table_stride=ts)
    check_embed_grad(ids, grad.expand(n, dim) if gs == 0 else grad, vocab, dim, 0.75, base, table, table_type)
    assert marks_untouched(whole, vocab, dim, ts, shift)


@pytest.mark.gpu
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("grad_type,table_type", [("f32", "bf16"), ("f32", "f16"), ("bf16", "f16"), ("f16", "bf16")])
@pytest.mark.parametrize("n,vocab,dim,gs,ts,shift,kind", GRAD_CASES)
def test_embed_grad_of_mixed_types(tok, grad_type, table_type, n, vocab, dim, gs, ts, shift, kind, accumulate):
    run_embed_grad(tok, grad_type, table_type, n, vocab, dim, gs, ts, shift, kind, accumulate)


@pytest.mark.gpu
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("grad_type,table_type", [("f32", "f32"), ("bf16", "f32"), ("f16", "f16"), ("f32", "bf16")])
@pytest.mark.parametrize("kind", ["one", "text", "wrong"])
@pytest.mark.parametrize("dim,shift", [(2051, 1), (4099, 1), (4099, 3), (1021, 0), (4104, 0), (8200, 0)])
def test_embed_grad_of_several_slabs(tok, grad_type, table_type, kind, dim, shift, accumulate):
    """More columns than a CTA takes at once, at any alignment, with sums of one block, of two and of many."""
    run_embed_grad(tok, grad_type, table_type, 523, 150, dim, dim, dim + (8 if shift == 0 else 5), shift, kind, accumulate)


@pytest.mark.gpu
@pytest.mark.parametrize("n,vocab,dim", [(70000, 300, 64), (150000, 50257, 40), (300000, 200000, 24), (1 << 20, 1 << 19, 8)])
@pytest.mark.parametrize("kind", ["text", "one", "all"])
def test_embed_grad_of_many_tokens(tok, n, vocab, dim, kind):
    import torch

    g = torch.Generator(device="cuda").manual_seed(n)
    grad = torch.randn(n, dim, generator=g, device="cuda")
    ids = some_ids(n, n, vocab, kind)
    table = torch.empty(vocab, dim, device="cuda")
    work = embed_grad(tok, ids, grad, "f32", vocab, dim, table, "f32", spare=4096)
    check_embed_grad(ids, grad, vocab, dim, 1.0, None, table, "f32")
    assert bool((work[-4096:] == 0xAB).all())


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 13, 101, 1003])
@pytest.mark.parametrize("dim", [16, 23])
def test_embed_grad_with_owners_that_have_no_token(tok, n, dim):
    """All ids in the lowest of the 128 residue classes that the tokens are dealt out by; no whole number of blocks."""
    import torch

    vocab = 1000
    ids = (some_ids(n, n, 7, "text") * 128 + some_ids(n + 1, n, 5, "text")).clamp(max=vocab - 1).to(torch.int32)
    grad = torch.randn(n, dim, device="cuda")
    table = torch.full((vocab, dim), 3.0, device="cuda")
    embed_grad(tok, ids, grad, "f32", vocab, dim, table, "f32")
    check_embed_grad(ids, grad, vocab, dim, 1.0, None, table, "f32")


@pytest.mark.gpu
def test_embed_grad_of_nothing(tok):
    import torch

    table = torch.full((5, 24), 3.0, device="cuda")
    tok.embed_grad(0, 0, 0, "f32", 5, 20, table.data_ptr(), "f32", 0, 0, accumulate=True, table_stride=24)
    assert bool((table == 3).all())
    tok.embed_grad(0, 0, 0, "f32", 5, 20, table.data_ptr(), "f32", 0, 0, table_stride=24)
    assert bool((table[:, :20] == 0).all()) and bool((table[:, 20:] == 3).all())


# ---------------------------------------------------------------------------------------------------- log probabilities
def some_logits(seed, n, vocab, kind):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, vocab, generator=g, device="cuda") * 3
    if kind == "masked":             # rows with fewer and fewer columns left, the last with none
        for r in range(n):
            allowed = torch.rand(vocab, generator=g, device="cuda") < 0.5 ** (1 + r % 12)
            x[r, ~allowed] = -math.inf
        x[n - 1] = -math.inf
    if kind == "lowest":             # masked with the type's lowest value; a whole row of it
        x[:, ::2] = -65504.0
        x[n // 2] = -65504.0
    if kind == "ties":               # few different values, a constant row
        x = x.round()
        x[n // 2] = 1.0
        x[0, ::3] = -0.0
        x[0, 1::3] = 0.0
    if kind == "peaked":             # far apart
        x = x * 30
    if kind == "rising":             # each column above the one before
        x = torch.arange(vocab, device="cuda").float().expand(n, vocab) / 64
    if kind == "crowded":            # the highest lie in columns that a few threads own
        x[:, torch.arange(vocab, device="cuda") % 2048 < 160] += 40
    return x


def score(tok, x, name, targets, k, scale, stride):
    import torch

    n, vocab = x.shape
    f = lambda *s: torch.full(s, 9.25, device="cuda")  # noqa: E731
    lp, H, lse, ids, tops = f(n + 1), f(n + 1), f(n + 1), torch.full((n * k + 1,), 77, device="cuda", dtype=torch.int32), f(n * k + 1)
    tok.token_logprobs(x.data_ptr(), name, n, vocab, targets.data_ptr(), lp.data_ptr(), H.data_ptr(), lse.data_ptr(), k,
                       ids.data_ptr() if k else 0, tops.data_ptr() if k else 0, scale=scale, stride=stride)
    for t in (lp, H, lse, tops):
        assert float(t[-1]) == 9.25
    assert int(ids[-1]) == 77
    return lp[:-1], H[:-1], lse[:-1], ids[:-1].view(n, k), tops[:-1].view(n, k)


def score_wanted(x, targets, k, scale):
    """Formulas in 64 bits and bounds: lists (value, bound)."""
    import torch

    n, vocab = x.shape
    scale = float(np.float32(scale))
    raw = x.double()
    top = raw.amax(1)
    none = top == -math.inf
    m = torch.where(none, torch.zeros_like(top), top)
    y = (raw - m[:, None]) * scale
    s = y.exp().sum(1)
    log_s = s.log()
    lse = m * scale + log_s
    logp = y - log_s[:, None]            # not z - lse: around the lowest number 64 bits hold no log_s
    logp[none] = -math.inf
    p = logp.exp()
    p[none] = 0
    H = torch.where(p > 0, -p * logp, torch.zeros_like(p)).sum(1)
    yy = torch.where(p > 0, p * y * y, torch.zeros_like(p)).sum(1)
    # y: three roundings; 2^y: the approximation's 2^-22 and y's error; every thread adds at most vocab / 256 + 8 numbers, the threads' sums
    # are joined in 13 steps with three roundings each, and a sum is rescaled (three roundings) once per new maximum of a
    # thread, 24 at the outside for columns in any order but a rising one, where they are as many as the columns
    steps = (vocab / 256 + 8) * 4 + 64
    rel = steps * U + 2.0 ** -22 + 4 * U * H
    lse_bound = rel + 2 * U * log_s.abs() + 2 * U * (m * scale).abs() + 2 * U * lse.abs()
    H_bound = rel * (2 * H + 2) + 8 * U * yy + 4 * U * log_s.abs()
    t = targets.long()
    inside = (t >= 0) & (t < vocab)
    lp = logp.gather(1, torch.where(inside, t, torch.zeros_like(t))[:, None])[:, 0]
    yt = y.gather(1, torch.where(inside, t, torch.zeros_like(t))[:, None])[:, 0]
    lp_bound = rel + 2 * U * log_s.abs() + 4 * U * torch.where(yt > -math.inf, yt.abs(), torch.zeros_like(yt))
    lp = torch.where(none & inside, torch.full_like(lp, -math.inf), lp)
    lp = torch.where(t < 0, torch.zeros_like(lp), torch.where(t >= vocab, torch.full_like(lp, math.nan), lp))
    order = torch.sort(raw, dim=1, descending=True, stable=True)
    best, ids = order.values[:, :k], order.indices[:, :k]
    if vocab < k:
        pad = torch.full((n, k - vocab), -1, device="cuda", dtype=ids.dtype)
        best, ids = torch.cat([best, pad.double() * math.inf], 1), torch.cat([ids, pad], 1)
    dead = best == -math.inf
    ids = torch.where(dead, torch.full_like(ids, -1), ids)
    tops = torch.where(dead, best, (best - m[:, None]) * scale - log_s[:, None])
    bt = torch.where(dead, torch.zeros_like(best), (best - m[:, None]).abs() * scale)
    tops_bound = (rel + 2 * U * log_s.abs())[:, None] + 4 * U * bt
    lse = torch.where(none, torch.full_like(lse, -math.inf), lse)
    return (lp, lp_bound), (H, H_bound), (lse, lse_bound), ids, (tops, tops_bound)


def same(got, want, bound, what):
    import torch

    got = got.double()
    assert bool((torch.isnan(got) == torch.isnan(want)).all()), what
    fine = torch.isfinite(want)
    assert bool((got[~fine & ~torch.isnan(want)] == want[~fine & ~torch.isnan(want)]).all()), what
    bound = bound.expand_as(want)[fine]
    err = (got[fine] - want[fine]).abs() - bound
    assert not bool((err > 0).any()), (what, float(err.max()), float(bound.max()))


SCORE_CASES = [
    (1, 1, 1, 0, "plain"), (3, 2, 2, 0, "plain"), (1, 50257, 50257, 0, "plain"), (5, 31, 40, 1, "masked"), (9, 257, 257, 0, "plain"),
    (20, 1000, 1000, 0, "masked"), (17, 1001, 1001, 1, "masked"), (4, 4099, 4104, 0, "ties"), (7, 8192, 8192, 0, "lowest"),
    (3, 50257, 50304, 0, "masked"), (2, 50257, 50257, 1, "ties"), (6, 32003, 32003, 3, "peaked"), (2, 131072, 131072, 0, "plain"),
    (2, 200001, 200001, 1, "masked"), (40, 3001, 3001, 0, "crowded"), (11, 50257, 50257, 0, "crowded"), (4, 9999, 9999, 0, "rising"),
    (160, 777, 777, 0, "masked"), (400, 2053, 2056, 5, "ties"), (1300, 513, 513, 0, "plain"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("n,vocab,stride,shift,kind", SCORE_CASES)
def test_token_logprobs(tok, name, n, vocab, stride, shift, kind):
    import torch

    _, x = rows(some_logits(n + vocab, n, vocab, kind), name, stride, shift)
    if kind == "lowest":
        lowest = torch.finfo(dtype(name)).min
        x[x == torch.tensor(-65504.0).to(dtype(name)).item()] = lowest
    targets = some_ids(vocab, n, vocab, "wrong" if n > 4 else "text")
    for k, scale in ((0, 1.0), (1, 0.7), (20, 1.0), (32, 1.3)):
        if kind == "lowest":
            scale = min(scale, 1.0)      # 1.3 times the lowest number of 32 bits is none
        lp, H, lse, ids, tops = score(tok, x, name, targets, k, scale, stride)
        w_lp, w_H, w_lse, w_ids, w_tops = score_wanted(x, targets, k, scale)
        assert torch.equal(ids.long(), w_ids), (k, scale)
        same(lse, *w_lse, "lse")
        same(lp, *w_lp, "logprob")
        same(H, *w_H, "entropy")
        same(tops, *w_tops, "top")


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [5, 1000, 50257])
def test_rows_without_a_distribution(tok, vocab):
    import torch

    x = some_logits(1, 6, vocab, "plain")
    x[1, vocab // 2] = math.nan
    x[2, vocab - 1] = math.inf
    x[3, 0] = math.nan
    x[3, 1:] = -math.inf
    x[4] = -math.inf
    targets = torch.tensor([1, 0, 2, -1, 3, vocab], device="cuda", dtype=torch.int32)
    lp, H, lse, ids, tops = score(tok, x, "f32", targets, 3, 1.0, vocab)
    for r in (1, 2, 3):
        assert math.isnan(lse[r]) and math.isnan(H[r]) and bool(torch.isnan(tops[r]).all()) and ids[r].tolist() == [-1] * 3
    assert math.isnan(lp[1]) and math.isnan(lp[2]) and float(lp[3]) == 0 and math.isnan(lp[5])
    assert float(lp[4]) == -math.inf and float(H[4]) == 0 and float(lse[4]) == -math.inf and ids[4].tolist() == [-1] * 3
    for r in (0, 5):
        assert bool(torch.isfinite(lse[r])) and (ids[r] >= 0).all()
    g = torch.ones(6, device="cuda")
    out = torch.full_like(x, 5.0)
    tok.token_logprobs_grad(x.data_ptr(), "f32", 6, vocab, targets.data_ptr(), lse.data_ptr(), g.data_ptr(), out.data_ptr())
    assert bool(torch.isnan(out[1]).all()) and bool((out[3:] == 0).all()) and bool(torch.isfinite(out[0]).all())


@pytest.mark.gpu
def test_outputs_that_are_not_wanted(tok):
    import torch

    x = some_logits(3, 5, 777, "plain")
    targets = some_ids(3, 5, 777, "text")
    lp, H, lse, ids, tops = score(tok, x, "f32", targets, 4, 1.0, 777)
    one = torch.full((5,), 9.0, device="cuda")
    tok.token_logprobs(x.data_ptr(), "f32", 5, 777, d_lse=one.data_ptr())
    assert torch.equal(one, lse)
    tok.token_logprobs(x.data_ptr(), "f32", 5, 777, d_entropy=one.data_ptr())
    assert torch.equal(one, H)
    tok.token_logprobs(x.data_ptr(), "f32", 5, 777, targets.data_ptr(), one.data_ptr())
    assert torch.equal(one, lp)
    few = torch.zeros(5, 4, device="cuda", dtype=torch.int32)
    tok.token_logprobs(x.data_ptr(), "f32", 5, 777, top_k=4, d_top_ids=few.data_ptr())
    assert torch.equal(few, ids)
    some = torch.zeros(5, 4, device="cuda")
    tok.token_logprobs(x.data_ptr(), "f32", 5, 777, top_k=4, d_top_logprobs=some.data_ptr())
    assert torch.equal(some, tops)
    tok.token_logprobs(0, "f32", 0, 777)
    same_row = x[2:3]
    tok.token_logprobs(same_row.data_ptr(), "f32", 5, 777, d_lse=one.data_ptr(), stride=0)
    assert bool((one == lse[2]).all())


def grad_wanted(x, targets, scale, g, e):
    """The gradient in 64 bits and a bound on what 32 bits and the given statistics' own rounding make of it."""
    import torch

    n, vocab = x.shape
    scale = float(np.float32(scale))
    z = x.double() * scale
    lse = torch.logsumexp(z, 1)
    none = lse == -math.inf
    safe = torch.where(none, torch.zeros_like(lse), lse)
    logp = z - safe[:, None]
    p = torch.where(none[:, None], torch.zeros_like(z), logp.exp())
    logp = torch.where(p > 0, logp, torch.zeros_like(logp))
    H = -(p * logp).sum(1)
    t = targets.long()
    inside = (t >= 0) & (t < vocab) & ~none
    g = torch.where(inside, g.double(), torch.zeros_like(g.double())) if g is not None else torch.zeros(n, device="cuda", dtype=torch.float64)
    here = (torch.arange(vocab, device="cuda")[None] == t[:, None]) & inside[:, None]
    d = g[:, None] * (here.double() - p)
    e = e.double() if e is not None else torch.zeros_like(g)
    inner = logp + H[:, None]
    d = d - e[:, None] * p * inner
    err_z = 3 * U * logp.abs() + 2 * U * safe.abs()[:, None]
    rel_p = err_z + 2.0 ** -22
    bound = p * rel_p * (g[:, None].abs() + (e[:, None] * inner).abs()) + e[:, None].abs() * p * (err_z + 4 * U * H[:, None] + 4 * U * inner.abs())
    # a p below 2^-126 (log p < -87) may count as 0: its whole part of the gradient, (|g| + |e (log p + H)|) p, is then missing
    logp = torch.where(none[:, None], torch.zeros_like(z), z - safe[:, None]).clamp(min=-1000)
    gone = p.clamp(max=2.0 ** -126) * (g[:, None].abs() + (e[:, None] * (logp + H[:, None])).abs())
    bound = bound + gone + 4 * U * (g[:, None].abs() * (here.double() + p) + (e[:, None] * p * inner).abs())
    return lse, H, d * scale, bound * scale


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("n,vocab,stride,shift,kind", [c for c in SCORE_CASES if c[4] != "lowest"])
@pytest.mark.parametrize("parts", ["logprob", "entropy", "both"])
def test_token_logprobs_grad(tok, name, n, vocab, stride, shift, kind, parts):
    import torch

    x_all, x = rows(some_logits(n + vocab, n, vocab, kind), name, stride, shift)
    targets = some_ids(vocab, n, vocab, "wrong" if n > 4 else "text")
    gen = torch.Generator(device="cuda").manual_seed(n)
    g = torch.randn(n, generator=gen, device="cuda") if parts != "entropy" else None
    e = torch.randn(n, generator=gen, device="cuda") if parts != "logprob" else None
    scale = 0.9
    lse, H, want, bound = grad_wanted(x, targets, scale, g, e)
    lse32, H32 = lse.float(), H.float()
    bound = bound + want.abs() * half_step(name) * 1.01 + tiny(name) + 1e-36

    def call(out, out_stride):
        tok.token_logprobs_grad(x.data_ptr(), name, n, vocab, targets.data_ptr() if g is not None else 0, lse32.data_ptr(),
                                g.data_ptr() if g is not None else 0, out.data_ptr(), H32.data_ptr() if e is not None else 0,
                                e.data_ptr() if e is not None else 0, scale=scale, stride=stride, grad_stride=out_stride)

    for out_stride, out_shift in ((stride, shift), (vocab + 3, 2), (stride, shift + 1)):
        whole, out = rows(torch.zeros(n, vocab, device="cuda"), name, out_stride, out_shift)
        call(out, out_stride)
        same(out, want, bound, (out_stride, out_shift))
        assert marks_untouched(whole, n, vocab, out_stride, out_shift)
    if stride >= vocab:
        call(x, stride)                                   # in place
        same(x, want, bound, "in place")
        assert marks_untouched(x_all, n, vocab, stride, shift)


@pytest.mark.gpu
def test_gradients_against_differences(tok):
    """Central differences of the formulas in 64 bits: their own error is h^2 / 6 times third derivatives below 8 here, and
    1e-16 / h of rounding times values below 4."""
    import torch

    n, vocab, scale = 4, 37, 0.8
    x = some_logits(5, n, vocab, "plain")
    targets = torch.tensor([0, 5, 36, -1], device="cuda", dtype=torch.int32)
    g = torch.tensor([1.0, -0.5, 2.0, 3.0], device="cuda")
    e = torch.tensor([0.5, 1.0, -1.0, 0.25], device="cuda")

    def value(v):
        z = v * float(np.float32(scale))
        logp = z - torch.logsumexp(z, 1, keepdim=True)
        lp = torch.where(targets >= 0, logp.gather(1, targets.clamp(min=0).long()[:, None])[:, 0], torch.zeros(n, device="cuda", dtype=torch.float64))
        return g.double() * lp - e.double() * (logp.exp() * logp).sum(1)

    h, want = 1e-4, torch.zeros(n, vocab, device="cuda", dtype=torch.float64)
    for c in range(vocab):
        d = torch.zeros_like(want)
        d[:, c] = h
        want[:, c] = (value(x.double() + d) - value(x.double() - d)) / (2 * h)
    _, H, lse, _, _ = score(tok, x, "f32", targets, 0, scale, vocab)
    out = torch.empty_like(x)
    tok.token_logprobs_grad(x.data_ptr(), "f32", n, vocab, targets.data_ptr(), lse.data_ptr(), g.data_ptr(), out.data_ptr(), H.data_ptr(),
                            e.data_ptr(), scale=scale)
    _, _, _, bound = grad_wanted(x, targets, scale, g, e)
    # the statistics come from the operator itself here: their error (of the order of 2^-20) counts too
    assert bool(((out.double() - want).abs() <= bound + 2.0 ** -20 * 4 + 8 * h * h + 4e-16 / h * 4).all())


# ---------------------------------------------------------------------------------------------------- as they are used
@pytest.mark.gpu
def test_from_text_to_gradients(native_built, merges_path):
    """Text on the device -> ids -> rows -> logits of a tied table -> log probabilities and alternatives -> text; and back:
    the gradient of the logits, and the table's from both its uses, against differentiation in 64 bits."""
    import torch

    import gputok_b200

    t = Tokenizer(merges_path, 1 << 16, 50, device=0)
    t.set_stream(torch.cuda.current_stream().cuda_stream)
    vocab, dim = 50257, 64
    data = gputok_b200.TextGen(3).text(3000)
    d_bytes = torch.from_numpy(data.copy()).cuda()
    d_off = torch.tensor([0, len(data)], dtype=torch.int64, device="cuda")
    ids = torch.empty(len(data), dtype=torch.int32, device="cuda")
    n, _, _ = t.encode_device(d_bytes.data_ptr(), len(data), d_off.data_ptr(), 1, ids.data_ptr(), len(data))
    ids = ids[:n]
    assert n > 300
    g = torch.Generator(device="cuda").manual_seed(1)
    table = torch.randn(vocab, dim, generator=g, device="cuda") * 0.3
    mix = torch.randn(dim, dim, generator=g, device="cuda") * 0.3
    x = torch.empty(n - 1, dim, device="cuda")
    t.embed(ids.data_ptr(), n - 1, table.data_ptr(), "f32", vocab, dim, x.data_ptr(), "f32", scale=8.0)
    hidden = (x.double() @ mix.double()).float()
    logits = (hidden.double() @ table.double().T).float()
    nxt = ids[1:].contiguous()
    lp, H, lse, tops, top_lps = score(t, logits, "f32", nxt, 5, 1.0, vocab)
    words = t.decode(tops.cpu().numpy().reshape(-1))
    assert len(words) >= 5 * (n - 1)
    assert t.decode(ids.cpu().numpy()) == data.tobytes()
    w = torch.full((n - 1,), -1.0 / (n - 1), device="cuda")    # mean loss
    t.token_logprobs_grad(logits.data_ptr(), "f32", n - 1, vocab, nxt.data_ptr(), lse.data_ptr(), w.data_ptr(), logits.data_ptr())
    d_table = logits.double().T @ hidden.double()              # the head's part
    d_x = ((logits.double() @ table.double()) @ mix.double().T).float()
    d_table = d_table.float()
    embed_grad(t, ids[:n - 1], d_x, "f32", vocab, dim, d_table, "f32", scale=8.0, accumulate=True)

    T = table.double().requires_grad_()
    z = (T[ids[:n - 1].long()] * 8.0 @ mix.double()) @ T.T
    logp = torch.log_softmax(z, 1)
    loss = -logp.gather(1, nxt.long()[:, None]).mean()
    loss.backward()
    assert abs(float(-lp.double().mean()) - float(loss)) < 1e-4
    # f32 logits of size up to 60 are off by 2e-6, their probabilities by as much, sums of products with numbers below 60 of them
    scale = float(T.grad.abs().max())
    assert float((d_table.double() - T.grad).abs().max()) < 1e-4 * scale


@pytest.mark.gpu
def test_captured_and_replayed(native_built, merges_path):
    """All four in one graph, replayed on other inputs in the same places; the handle's first calls of them."""
    import torch

    t = Tokenizer(merges_path, 2048, 50, device=0)
    n, vocab, dim = 3000, 1000, 96
    s = torch.cuda.Stream()
    ids = some_ids(1, n, vocab, "padded")
    table = torch.randn(vocab, dim, device="cuda")
    out = torch.empty(n, dim, device="cuda")
    grad = torch.empty(vocab, dim, device="cuda")
    logits = some_logits(2, n, vocab, "plain")
    lp, H, lse = (torch.empty(n, device="cuda") for _ in range(3))
    top = torch.empty(n, 5, device="cuda", dtype=torch.int32)
    w = torch.randn(n, device="cuda")
    d_logits = torch.empty(n, vocab, device="cuda")
    work = torch.empty(t.embed_grad_workspace(n, vocab, dim), device="cuda", dtype=torch.uint8)

    def calls():
        t.embed(ids.data_ptr(), n, table.data_ptr(), "f32", vocab, dim, out.data_ptr(), "f32")
        t.token_logprobs(logits.data_ptr(), "f32", n, vocab, ids.data_ptr(), lp.data_ptr(), H.data_ptr(), lse.data_ptr(), 5, top.data_ptr())
        t.token_logprobs_grad(logits.data_ptr(), "f32", n, vocab, ids.data_ptr(), lse.data_ptr(), w.data_ptr(), d_logits.data_ptr())
        t.embed_grad(ids.data_ptr(), n, out.data_ptr(), "f32", vocab, dim, grad.data_ptr(), "f32", work.data_ptr(), work.numel())

    torch.cuda.synchronize()
    t.set_stream(s.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        calls()
    results = (out, grad, lp, H, lse, top, d_logits)
    for seed in (4, 5):
        ids.copy_(some_ids(seed, n, vocab, "padded"))
        logits.copy_(some_logits(seed, n, vocab, "plain"))
        work.fill_(0x55)
        for r in results:
            r.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        got = [r.clone() for r in results]
        for r in results:
            r.fill_(4)
        torch.cuda.synchronize()
        calls()
        torch.cuda.synchronize()
        for a, b in zip(got, results):
            assert torch.equal(a.nan_to_num(nan=-5.0), b.nan_to_num(nan=-5.0))
        check_embed_grad(ids, out, vocab, dim, 1.0, None, grad, "f32")


@pytest.mark.gpu
def test_two_handles_on_two_streams(native_built, merges_path):
    """Calls of two handles at once, each with its own workspace, give what they give alone."""
    import torch

    n, vocab, dim = 20000, 5000, 128
    a, b = (Tokenizer(merges_path, 2048, 50, device=0) for _ in range(2))
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    a.set_stream(sa.cuda_stream)
    b.set_stream(sb.cuda_stream)
    sets = []
    for t, seed in ((a, 1), (b, 2)):
        ids = some_ids(seed, n, vocab, "text")
        grad = torch.randn(n, dim, device="cuda")
        sets.append((t, ids, grad, torch.empty(vocab, dim, device="cuda"),
                     torch.empty(t.embed_grad_workspace(n, vocab, dim), device="cuda", dtype=torch.uint8)))
    torch.cuda.synchronize()
    for _ in range(5):
        for t, ids, grad, out, work in sets:
            t.embed_grad(ids.data_ptr(), n, grad.data_ptr(), "f32", vocab, dim, out.data_ptr(), "f32", work.data_ptr(), work.numel())
    torch.cuda.synchronize()
    for t, ids, grad, out, work in sets:
        check_embed_grad(ids, grad, vocab, dim, 1.0, None, out, "f32")


@pytest.mark.gpu
def test_offsets_beyond_32_bits(tok):
    """A table and rows of logits whose last elements lie more than 2^32 elements behind the first."""
    import torch

    vocab, dim, n = 40, 16, 6
    stride = 1 << 27
    table = torch.empty(39 * stride + dim, device="cuda", dtype=torch.bfloat16)   # 10 GiB, hardly any of it touched
    view = table.as_strided((vocab, dim), (stride, 1))
    view.copy_(torch.randn(vocab, dim, device="cuda"))
    ids = torch.tensor([39, 0, 38, 33, 39, 32], device="cuda", dtype=torch.int32)
    out = torch.empty(n, dim, device="cuda")
    tok.embed(ids.data_ptr(), n, view.data_ptr(), "bf16", vocab, dim, out.data_ptr(), "f32", table_stride=stride)
    assert torch.equal(out, view[ids.long()].float())
    grad = torch.randn(n, dim, device="cuda")
    embed_grad(tok, ids, grad, "f32", vocab, dim, view, "bf16", table_stride=stride)
    check_embed_grad(ids, grad, vocab, dim, 1.0, None, view, "bf16")
    view.copy_(torch.randn(vocab, dim, device="cuda"))
    targets = some_ids(1, vocab, dim, "text")
    lp, H, lse, top, tops = score(tok, view, "bf16", targets, 3, 1.0, stride)
    w_lp, w_H, w_lse, w_ids, w_tops = score_wanted(view, targets, 3, 1.0)
    assert torch.equal(top.long(), w_ids)
    same(lp, *w_lp, "logprob")
    ones = torch.ones(vocab, device="cuda")
    _, _, want, bound = grad_wanted(view, targets, 1.0, ones, None)
    tok.token_logprobs_grad(view.data_ptr(), "bf16", vocab, dim, targets.data_ptr(), lse.data_ptr(), ones.data_ptr(), view.data_ptr(),
                            stride=stride, grad_stride=stride)
    same(view, want, bound + 2.0 ** -20 + want.abs() * half_step("bf16") * 1.01, "in place")


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [0, 1, 2, 3])
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 127, 1023, 1025, 70001])
def test_ids_at_any_address(tok, n, shift):
    """The ids are read sixteen bytes at a time: first and last ones that share these with strangers."""
    import torch

    vocab, dim = 500, 12
    whole = torch.full((n + 16,), 3, device="cuda", dtype=torch.int32)   # strangers that would be ids
    ids = whole[shift + 4:shift + 4 + n]
    ids.copy_(some_ids(n, n, vocab, "padded"))
    grad = torch.randn(n, dim, device="cuda")
    table = torch.empty(vocab, dim, device="cuda")
    embed_grad(tok, ids, grad, "f32", vocab, dim, table, "f32")
    check_embed_grad(ids, grad, vocab, dim, 1.0, None, table, "f32")


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [24, 23, 136])
@pytest.mark.parametrize("n", [700, 5000, 40000, 150000])
def test_sums_of_every_length(tok, n, dim):
    """Ids that occur once, twice, .. and the rest on one id, so that sums begin and end at all places of the blocks that the
    tokens are dealt with in."""
    import torch

    counts, left = [], n
    while left > 0:
        counts.append(min(left, 1 + len(counts) % 150))
        left -= counts[-1]
    vocab = len(counts) + 200
    g = torch.Generator().manual_seed(n)
    ids = torch.repeat_interleave(torch.randperm(vocab, generator=g)[:len(counts)], torch.tensor(counts))
    ids = ids[torch.randperm(n, generator=g)].to(torch.int32).cuda()
    for name in ("f32", "bf16"):
        _, grad = rows(torch.randn(n, dim, device="cuda"), name)
        table = torch.empty(vocab, dim, device="cuda")
        embed_grad(tok, ids, grad, name, vocab, dim, table, "f32")
        check_embed_grad(ids, grad, vocab, dim, 1.0, None, table, "f32")
        base = table.clone()
        embed_grad(tok, ids, grad, name, vocab, dim, table, "f32", accumulate=True)
        check_embed_grad(ids, grad, vocab, dim, 1.0, base, table, "f32")


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("n,vocab,stride,shift,kind", [
    (800, 9001, 9001, 0, "masked"), (1500, 7001, 7001, 1, "ties"), (900, 12288, 12288, 0, "crowded"), (2000, 100, 104, 0, "masked"),
    (760, 20011, 20016, 0, "lowest"), (30, 70001, 70001, 0, "rising"), (64, 100003, 100003, 1, "ties"), (12, 131072, 131072, 0, "crowded"),
])
def test_token_logprobs_of_other_shapes(tok, name, n, vocab, stride, shift, kind):
    """More rows than a wave of CTAs, and rows that several CTAs share, against the same bounds."""
    import torch

    _, x = rows(some_logits(n + vocab, n, vocab, kind), name, stride, shift)
    if kind == "lowest":
        x[x == torch.tensor(-65504.0).to(dtype(name)).item()] = torch.finfo(dtype(name)).min
    targets = some_ids(vocab, n, vocab, "wrong")
    for k in (0, 3, 32):
        lp, H, lse, ids, tops = score(tok, x, name, targets, k, 1.0, stride)
        w_lp, w_H, w_lse, w_ids, w_tops = score_wanted(x, targets, k, 1.0)
        assert torch.equal(ids.long(), w_ids), k
        same(lse, *w_lse, "lse")
        same(lp, *w_lp, "logprob")
        same(H, *w_H, "entropy")
        same(tops, *w_tops, "top")


@pytest.mark.gpu
def test_the_same_bits_every_time(tok):
    import torch

    n, vocab, dim = 30000, 20000, 200
    ids = some_ids(3, n, vocab, "padded")
    grad = torch.randn(n, dim, device="cuda")
    first = None
    for _ in range(4):
        table = torch.empty(vocab, dim, device="cuda")
        embed_grad(tok, ids, grad, "f32", vocab, dim, table, "f32")
        first = table if first is None else first
        assert torch.equal(first, table)
    x = some_logits(9, 300, vocab, "ties")
    targets = some_ids(9, 300, vocab, "text")
    want = score(tok, x, "f32", targets, 20, 0.7, vocab)
    for _ in range(4):
        for a, b in zip(want, score(tok, x, "f32", targets, 20, 0.7, vocab)):
            assert torch.equal(a, b)


def test_scales_that_32_bits_do_not_hold(host):
    for scale in (1.1e38, 3e38, 5e-324):
        for name, good in (("token_logprobs", SCORE), ("token_logprobs_grad", SCORE_GRAD)):
            with pytest.raises(GtkError) as e:
                getattr(host, name)(**good, scale=scale)
            assert e.value.code == 1


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-38, 1e-20, 1e20, 1e38])
def test_scales_at_the_ends(tok, scale):
    """Logits of which the scale makes numbers around one."""
    import torch

    n, vocab = 6, 3001
    x = torch.randn(n, vocab, device="cuda") * 3
    x = (x.double() / scale).float() if scale > 1 else x * (0.1 / scale if scale > 1e-30 else 1e37)
    targets = some_ids(2, n, vocab, "text")
    lp, H, lse, ids, tops = score(tok, x, "f32", targets, 9, scale, vocab)
    w_lp, w_H, w_lse, w_ids, w_tops = score_wanted(x, targets, 9, scale)
    # the scale's product with log2(e), and logits below 2^-126, have their own steps: 2^-149 each, of numbers down to 1e-38
    more = 2.0 ** -149 / min(scale, 1e-37) * 16
    assert torch.equal(ids.long(), w_ids)
    same(lse, w_lse[0], w_lse[1] + more, "lse")
    same(lp, w_lp[0], w_lp[1] + more, "logprob")
    same(H, w_H[0], w_H[1] + more, "entropy")


@pytest.mark.gpu
def test_rows_of_many_millions(tok):
    """Rows that a CTA reads in more than 4096 batches, all rows being the same one, and one that CTAs share."""
    import torch

    vocab, k = 40_000_003, 20
    g = torch.Generator(device="cuda").manual_seed(5)
    x = (torch.randn(vocab, generator=g, device="cuda") * 0.25).to(torch.bfloat16)
    places = torch.randperm(vocab, generator=g, device="cuda")[:k]
    x[places] = torch.arange(2, 2 + k, device="cuda").to(torch.bfloat16)
    raw = x.double()
    lse = float(torch.logsumexp(raw, 0))
    p = (raw - lse).exp()
    H = float(-(p * (raw - lse)).sum())
    bound = (vocab / 256 + 8) * 4 * U + 2.0 ** -20           # see score_wanted
    for n in (1, 150):
        f = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
        lp, entropy, got_lse, top = f(n), f(n), f(n), torch.zeros(n, k, device="cuda", dtype=torch.int32)
        targets = torch.full((n,), vocab - 1, device="cuda", dtype=torch.int32)
        tok.token_logprobs(x.data_ptr(), "bf16", n, vocab, targets.data_ptr(), lp.data_ptr(), entropy.data_ptr(), got_lse.data_ptr(), k,
                           top.data_ptr(), stride=0)
        assert torch.equal(top.long(), places.flip(0).expand(n, k))
        assert bool(((got_lse.double() - lse).abs() < bound + 4 * U * lse).all())
        assert bool(((lp.double() - (float(raw[-1]) - lse)).abs() < bound + 8 * U * lse).all())
        assert bool(((entropy.double() - H).abs() < bound * (2 * H + 2) + 4 * U * lse).all())


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
def test_gradient_of_one_row_for_all(tok, name):
    """Logits with a stride of zero, which is not the gradient's."""
    import torch

    n, vocab = 700, 300
    ids = some_ids(4, n, vocab, "padded")
    _, x = rows(torch.randn(1, vocab, device="cuda"), name)
    g = torch.randn(n, device="cuda")
    lse, H, want, bound = grad_wanted(x.expand(n, vocab), ids, 1.0, g, None)
    lse32 = lse.float()
    for stride in (vocab, vocab + 4, vocab + 5):
        whole, grad = rows(torch.zeros(n, vocab, device="cuda"), name, stride)
        tok.token_logprobs_grad(x.data_ptr(), name, n, vocab, ids.data_ptr(), lse32.data_ptr(), g.data_ptr(), grad.data_ptr(), stride=0,
                                grad_stride=stride)
        same(grad, want, bound + want.abs() * half_step(name) * 1.01 + tiny(name) + 1e-36, "grad")
        assert marks_untouched(whole, n, vocab, stride, 0)


@pytest.mark.gpu
def test_two_threads_with_calls_of_different_sizes(native_built, merges_path):
    """A handle for each of two threads on one device, whose calls want different amounts of shared memory, above 48 KiB all of
    them: 2048 columns of 16 bits, sums in blocks of 8, 16 and 32 tokens."""
    import threading

    import torch

    vocab, dim = 300, 2048
    handles = [Tokenizer(merges_path, 2048, 50, device=0) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    work = [[], []]
    for i, sizes in enumerate(((2048,), (32768, 8192))):
        handles[i].set_stream(streams[i].cuda_stream)
        for n in sizes:
            grad = torch.randn(n, dim, device="cuda").to(torch.bfloat16)
            work[i].append((some_ids(n, n, vocab, "text"), grad, torch.empty(vocab, dim, device="cuda"),
                            torch.empty(handles[i].embed_grad_workspace(n, vocab, dim), device="cuda", dtype=torch.uint8)))
    torch.cuda.synchronize()
    start, failed = threading.Barrier(2), []

    def run(i):
        try:
            start.wait()
            for _ in range(2000 // len(work[i])):
                for ids, grad, table, space in work[i]:
                    handles[i].embed_grad(ids.data_ptr(), ids.numel(), grad.data_ptr(), "bf16", vocab, dim, table.data_ptr(), "f32",
                                          space.data_ptr(), space.numel())
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed
    for i in range(2):
        for ids, grad, table, _ in work[i]:
            check_embed_grad(ids, grad, vocab, dim, 1.0, None, table, "f32")


@pytest.mark.gpu
def test_a_failed_launch_is_the_calls_own(native_built, merges_path, oracle, novel):
    """A launch that CUDA refuses on the host (on the legacy stream while a stream that waits for it is being captured) is reported
    by its call, and by no later one."""
    import ctypes

    import torch

    t = Tokenizer(merges_path, 2048, 50, device=0)
    t.set_stream(0)
    ids = torch.tensor([3, 1], device="cuda", dtype=torch.int32)
    table, out = torch.randn(10, 8, device="cuda"), torch.full((2, 8), 5.0, device="cuda")
    torch.cuda.synchronize()
    want, _, _, _ = t.encode(novel[:5000])
    runtime = ctypes.CDLL("libcudart.so.12")         # another copy of the runtime than the one that the library holds
    stream, graph = ctypes.c_void_p(), ctypes.c_void_p()
    assert runtime.cudaStreamCreate(ctypes.byref(stream)) == 0
    assert runtime.cudaStreamBeginCapture(stream, 2) == 0
    try:
        with pytest.raises(GtkError) as e:
            t.embed(ids.data_ptr(), 2, table.data_ptr(), "f32", 10, 8, out.data_ptr(), "f32")
    finally:
        runtime.cudaStreamEndCapture(stream, ctypes.byref(graph))
        if graph:
            runtime.cudaGraphDestroy(graph)
        runtime.cudaStreamDestroy(stream)
        runtime.cudaGetLastError()
    assert e.value.code == 3 and "launch" in str(e.value)
    got, _, _, _ = t.encode(novel[:5000])
    assert np.array_equal(got, want)
    t.embed(ids.data_ptr(), 2, table.data_ptr(), "f32", 10, 8, out.data_ptr(), "f32")
    assert torch.equal(out, table[ids.long()])


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("vocab,shift", [(1000, 0), (4099, 0), (4099, 1)])
def test_rows_that_no_gradient_reaches(tok, name, vocab, shift):
    """Rows with both parts of their gradient zero (a loss mask, padding) get zeros whatever they and their statistics hold;
    a zero of one part alone takes nothing from the other."""
    import torch

    n, nan = 6, math.nan
    _, x = rows(some_logits(3, n, vocab, "plain"), name)
    targets = torch.tensor([1, 2, 3, -1, vocab, 4], device="cuda", dtype=torch.int32)
    g = torch.tensor([0.0, -0.0, 0.0, 3.0, nan, 1.0], device="cuda")
    e = torch.tensor([0.0, 0.0, 0.5, 0.0, -0.0, 0.0], device="cuda")
    lse, H, want, bound = grad_wanted(x, targets, 1.0, g, e)
    lse, H = lse.float(), H.float()
    for r in (1, 3, 4):                # what the padding of a batch may hold
        x[r] = nan
        x[r, ::2] = math.inf
        lse[r] = H[r] = nan
    bound = bound + want.abs() * half_step(name) * 1.01 + tiny(name) + 1e-36
    none = torch.tensor([0, 1, 3, 4], device="cuda")
    for entropy in (True, False):
        whole, out = rows(torch.ones(n, vocab, device="cuda"), name, vocab, shift)
        tok.token_logprobs_grad(x.data_ptr(), name, n, vocab, targets.data_ptr(), lse.data_ptr(), g.data_ptr(), out.data_ptr(),
                                H.data_ptr() if entropy else 0, e.data_ptr() if entropy else 0)
        assert bool((out[none] == 0).all()), entropy
        assert marks_untouched(whole, n, vocab, vocab, shift)
        same(out[5:], want[5:], bound[5:], "log probability alone")
        if entropy:
            same(out[2:3], want[2:3], bound[2:3], "entropy alone")
        else:
            assert bool((out[2] == 0).all())


def far_logits(seed, n, vocab, name, kind):
    """Rows whose log of the sum is large next to what tells their logits apart, in values of the type."""
    import torch

    t = dtype(name)
    x = some_logits(seed, n, vocab, "plain")
    if kind == "lowest":               # masked with the type's lowest value, every third row all of it
        x = x.to(t)
        x[:, ::2] = torch.finfo(t).min
        x[::3] = torch.finfo(t).min
        return x
    if kind == "highest":              # every third row at the other end, scale times which is no 32-bit number; one of -inf
        x = x.to(t)
        x[::3] = torch.finfo(t).max
        x[1::3] = torch.finfo(t).min
        x[1, ::3] = -math.inf
        x[n - 1] = -math.inf
        return x
    if kind == "masked":
        x[:, 1::3] = -math.inf
        x[n // 2] = -math.inf
    return (x + {"up": 3e4, "masked": -2e4, "down": -1e3}[kind]).to(t)


def grad_from_maximum(x, targets, scale, g, e, H, H_err):
    """grad_wanted() with log p_j = scale (x_j - m) - ln S in 64 bits, and a bound that is relative to p: of lse only what
    the header allows, 2^-24 of it below 256."""
    import torch

    n, vocab = x.shape
    scale = float(np.float32(scale))
    raw = x.double()
    top = raw.amax(1)
    none = top == -math.inf
    m = torch.where(none, torch.zeros_like(top), top)
    y = (raw - m[:, None]) * scale
    log_s = torch.where(none, torch.zeros_like(top), y.exp().sum(1).log())
    logp = y - log_s[:, None]
    p = torch.where(none[:, None], torch.zeros_like(y), logp.exp())
    y = y.clamp(min=-1e4)
    logp = logp.clamp(min=-1e4)
    lse = m * scale + log_s
    t = targets.long()
    inside = (t >= 0) & (t < vocab) & ~none
    zero = torch.zeros(n, device="cuda", dtype=torch.float64)
    g = zero if g is None else torch.where(inside, g.double(), zero)
    e = zero if e is None else e.double()
    here = (torch.arange(vocab, device="cuda")[None] == t[:, None]) & inside[:, None]
    inner = logp + H.double()[:, None]
    d = g[:, None] * (here.double() - p) - e[:, None] * p * inner
    # S as in score_wanted(); y and log p: a rounding of the difference, one of the product, one of the sum, and ln S's own three
    steps = (vocab / 256 + 8) * 4 + 64
    of_sum = steps * U + 2.0 ** -22 + 4 * U * (-(p * logp).sum(1)) + 3 * U * log_s.abs()
    of_lse = torch.where(lse.abs() < 256, 2 * U * lse.abs(), zero)
    err_z = (of_sum + of_lse)[:, None] + U * (2 * y.abs() + 3 * logp.abs())
    size = g[:, None].abs() + (e[:, None] * inner).abs()
    bound = p * (err_z + 2.0 ** -22) * size + e[:, None].abs() * p * (err_z + H_err[:, None] + 4 * U * inner.abs())
    bound = bound + p.clamp(max=2.0 ** -126) * (g[:, None].abs() + e[:, None].abs() * (inner.abs() + 1)) + 4 * U * (g[:, None].abs() * (here.double() + p) + (e[:, None] * p * inner).abs())
    return d * scale, bound * scale


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("kind,scale", [("lowest", 1.0), ("lowest", 0.7), ("lowest", 1.3), ("highest", 1.3), ("up", 1.0), ("masked", 0.9), ("down", 1.0)])
@pytest.mark.parametrize("n,vocab,stride,shift", [(3, 1000, 1000, 0), (5, 50257, 50257, 0), (7, 8193, 8200, 3), (700, 2053, 2056, 1), (2, 5, 5, 0)])
def test_gradient_where_the_sum_is_far_from_the_logits(tok, name, kind, scale, n, vocab, stride, shift):
    """The gradient from the statistics that token_logprobs gives for the same rows: 32 bits of lse say little about them."""
    import torch

    x_all, x = rows(far_logits(n + vocab, n, vocab, name, kind), name, stride, shift)
    targets = some_ids(vocab, n, vocab, "wrong" if n > 4 else "text")
    gen = torch.Generator(device="cuda").manual_seed(n)
    g, e = torch.randn(n, generator=gen, device="cuda"), torch.randn(n, generator=gen, device="cuda")
    _, H, lse, _, _ = score(tok, x, name, targets, 0, scale, stride)
    H_err = score_wanted(x, targets, 0, scale)[1][1]
    before = x.clone()
    for entropy in (False, True):
        want, bound = grad_from_maximum(before, targets, scale, g, e if entropy else None, H, H_err)
        bound = bound + want.abs() * half_step(name) * 1.01 + tiny(name) + 1e-36
        more = dict(d_entropy=H.data_ptr(), d_grad_entropy=e.data_ptr()) if entropy else {}
        for out_stride, out_shift in ((stride, shift), (stride + 1, shift + 1)):
            whole, out = rows(torch.ones(n, vocab, device="cuda"), name, out_stride, out_shift)
            tok.token_logprobs_grad(x.data_ptr(), name, n, vocab, targets.data_ptr(), lse.data_ptr(), g.data_ptr(), out.data_ptr(), scale=scale,
                                    stride=stride, grad_stride=out_stride, **more)
            same(out, want, bound, (entropy, out_stride))
            assert marks_untouched(whole, n, vocab, out_stride, out_shift)
    tok.token_logprobs_grad(x.data_ptr(), name, n, vocab, targets.data_ptr(), lse.data_ptr(), g.data_ptr(), x.data_ptr(), scale=scale, stride=stride,
                            grad_stride=stride, **more)
    same(x, want, bound, "in place")
    assert marks_untouched(x_all, n, vocab, stride, shift)


@pytest.mark.gpu
def test_checked_build_of_the_operators(native_built):
    """The library with index checks (-DGTK_CHECKED) through the small cases of this file, in a process of its own: no check of an
    index may fail.  Before that a check in either source file is made to fail, and is reported with its number, value and limit."""
    import os
    import subprocess
    import sys

    from gputok_b200.capi import checked_library_path

    path = checked_library_path()
    probe = ("import ctypes,sys; lib=ctypes.CDLL(sys.argv[1]); w=(ctypes.c_int*4)()\n"
             "for t in (2, 3, 0): print(lib.gtk_debug_check_words(w, 1, t), *w)")
    out = subprocess.run([sys.executable, "-c", probe, path], capture_output=True, text=True, timeout=300)
    assert out.stdout.split("\n")[:3] == ["0 299 5 4 1", "0 399 5 4 1", "0 0 0 0 0"], out.stdout + out.stderr
    chosen = ("(test_embed or test_sums or test_ids or owners or two_handles or captured or token_logprobs or rows_without or far_from or "
              "no_gradient) and not checked")
    run = subprocess.run([sys.executable, "-m", "pytest", os.path.abspath(__file__), "-m", "gpu", "-x", "-q", "-s", "-k", chosen],
                         capture_output=True, text=True, timeout=1500, env=dict(os.environ, GPUTOK_B200_LIBRARY=path))
    assert run.returncode == 0, run.stdout[-3000:] + run.stderr[-2000:]
    assert "CHECKED_BUILD rc=0 failures=0" in run.stdout, run.stdout[-2000:]


@pytest.mark.gpu
def test_measured_cases_follow_the_current_stream(native_built):
    """perf/operators.py: what is prepared under a stream runs on it, behind what the stream has in front, and goes into a graph that
    is captured from it, whichever stream was the first."""
    import importlib.util
    import os

    import torch

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf", "operators.py")
    spec = importlib.util.spec_from_file_location("perf_operators", path)
    ops = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ops)
    ops.own = True
    case = dict(ops._embed("embed", 200, 1000, 64, "f32", "f32"), name="small")
    first = ops.prepare(case, 1)
    ops.run(first)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        state = ops.prepare(case, 2)
        ops.run(state).fill_(0)
        torch.cuda._sleep(50_000_000)            # some 25 ms
        state["table"].mul_(2)
        out = ops.run(state)
        got = out.clone()
    torch.cuda.synchronize()
    want = state["table"][state["ids"].long()]
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        ops.run(state)
    state["table"].mul_(2)
    out.fill_(0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want * 2)
