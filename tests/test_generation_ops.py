"""A step of generation (blocks of a paged cache, slots of new tokens, ids drawn from logits) against plain implementations in
64 bits, through the C ABI.

Whole numbers are equal, but for ids where the definition's own comparison of two sums is closer than sums of 64-bit numbers in
another order are: a sum of n of them is off by at most (n - 1) 2^-53 of itself, a weight by a few 2^-53.
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

SAMPLE = dict(d_logits=P, type="f32", n_rows=3, vocab=10, d_uniform=P, d_ids=P, d_logprob=P, d_temperature=P, d_top_k=P, d_top_p=P,
              d_min_p=P)
TABLES = dict(d_old_lengths=P, d_new_lengths=P, n_requests=3, block_tokens=16, d_tables=P, columns=8, d_queue=P, queue_capacity=100,
              d_state=P, d_state_out=P)
SLOTS = dict(d_old_lengths=P, d_new_lengths=P, n_requests=3, block_tokens=16, d_tables=P, columns=8, capacity=20, d_slots=P, d_offsets=P,
             d_positions=P, d_requests=P, d_state=P)

REFUSED = [
    ("sample", SAMPLE, [dict(n_rows=-1), dict(vocab=0), dict(n_rows=1 << 31), dict(vocab=(1 << 20) + 1), dict(stride=-1), dict(d_logits=0),
                        dict(d_uniform=0), dict(d_ids=0), dict(d_logits=P + 2), dict(d_logits=P + 1, type="bf16"), dict(d_uniform=P + 4),
                        dict(d_ids=P + 2), dict(d_logprob=P + 1), dict(d_temperature=P + 2), dict(d_top_k=P + 2), dict(d_top_p=P + 3),
                        dict(d_min_p=P + 2)]),
    ("block_tables", TABLES, [dict(n_requests=-1), dict(n_requests=1 << 31), dict(block_tokens=0), dict(block_tokens=(1 << 20) + 1),
                              dict(columns=0), dict(columns=1 << 31), dict(table_stride=7), dict(queue_capacity=0), dict(queue_capacity=1 << 31),
                              dict(d_old_lengths=0), dict(d_new_lengths=0), dict(d_tables=0), dict(d_queue=0), dict(d_state=0),
                              dict(d_state_out=0), dict(d_old_lengths=P + 2), dict(d_new_lengths=P + 1), dict(d_tables=P + 2),
                              dict(d_queue=P + 2), dict(d_state=P + 4), dict(d_state_out=P + 4), dict(n_requests=0, d_state=0)]),
    ("slot_map", SLOTS, [dict(n_requests=-1), dict(n_requests=1 << 31), dict(block_tokens=0), dict(block_tokens=(1 << 20) + 1), dict(columns=0),
                         dict(columns=1 << 31), dict(table_stride=7), dict(capacity=-1), dict(capacity=1 << 31), dict(d_old_lengths=0),
                         dict(d_new_lengths=0), dict(d_tables=0), dict(d_slots=0), dict(d_offsets=0), dict(d_old_lengths=P + 2),
                         dict(d_new_lengths=P + 2), dict(d_tables=P + 1), dict(d_slots=P + 4), dict(d_offsets=P + 4), dict(d_positions=P + 2),
                         dict(d_requests=P + 2), dict(d_state=P + 4), dict(n_requests=0, d_offsets=0)]),
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
    assert lib.gtk_sample(host._h, P, 7, 1, 10, 10, P, None, None, None, None, P, None) == 1
    assert lib.gtk_sample(None, P, 0, 1, 10, 10, P, None, None, None, None, P, None) == 1
    assert lib.gtk_block_tables(None, P, P, 1, 16, P, 8, 8, P, 8, P, P) == 1
    assert lib.gtk_slot_map(None, P, P, 1, 16, P, 8, 8, None, 4, P, None, None, P) == 1


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


def rows(values, name, stride=None, shift=0):
    """The values (n x d) in an array of the type with a stride and a first element `shift` elements behind an aligned one;
    what lies around is NaN: nothing may be made of it."""
    import torch

    n, d = values.shape
    stride = d if stride is None else stride
    whole = torch.full(((n - 1) * stride + d + shift + 16,), math.nan, device="cuda", dtype=dtype(name))
    view = whole[shift:].as_strided((n, d), (stride, 1))
    view.copy_(values)
    return view


# ---------------------------------------------------------------------------------------------------- sampling
def some_logits(seed, n, vocab, kind):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, vocab, generator=g, device="cuda") * 2.5
    if kind in ("text", "masked", "lowest", "few"):  # a head of likely ids, whose lead differs from row to row
        at = torch.randint(0, vocab, (n, 40), generator=g, device="cuda")
        lead = 4 + 16 * torch.rand(n, 1, generator=g, device="cuda")
        x.scatter_add_(1, at, lead / (1 + 0.15 * torch.arange(40, device="cuda")))
    if kind == "equal":
        x.fill_(1.5)
    if kind == "ties":
        x = torch.randint(-3, 4, (n, vocab), generator=g, device="cuda").float() * 0.5
    if kind == "zeros":                              # both zeros, which are equal
        x = torch.where(torch.rand(n, vocab, generator=g, device="cuda") < 0.5, -0.0, 0.0)
    if kind == "rising":
        x = torch.linspace(-8, 8, vocab, device="cuda").expand(n, vocab).clone()
    if kind == "falling":
        x = torch.linspace(9, -30, vocab, device="cuda").expand(n, vocab).clone()
    if kind == "far":                                # a large common part, and one far above all others
        x += 3000.0
        x[:, vocab // 3] += 500.0
    if kind == "wide":                               # everything from -60000 to 60000
        x *= 8000.0
        x.clamp_(-60000.0, 60000.0)
    if kind == "masked":
        x[:, ::2] = -math.inf
    if kind == "lowest":                             # masks as the type's lowest number
        x[:, 1::3] = -math.inf                       # replaced in the type, see below
    if kind == "few":                                # a handful of columns is allowed
        keep = torch.randint(0, vocab, (n, 5), generator=g, device="cuda")
        y = torch.full_like(x, -math.inf)
        x = y.scatter_(1, keep, x.gather(1, keep))
    if kind == "one":
        y = torch.full_like(x, -math.inf)
        y[:, vocab - 1] = -40.0
        x = y
    return x


def typed_logits(seed, n, vocab, kind, name, stride=None, shift=0):
    import torch

    x = some_logits(seed, n, vocab, kind).to(dtype(name))
    if kind == "lowest":
        x = torch.where(torch.isneginf(x), torch.full_like(x, torch.finfo(dtype(name)).min), x)
    return rows(x, name, stride, shift)


def possible_draws(x, t, k, p, least, u):
    """[(id, log probability)] that the definition gives for a row: one, but where two sums meet to within what 64 bits hold."""
    if u < 0:
        return [(-1, 0.0)]
    if not (0 <= t < math.inf) or math.isnan(p) or math.isnan(least) or math.isnan(u) or np.isnan(x).any() or (x == math.inf).any():
        return [(-1, math.nan)]
    order = np.lexsort((np.arange(len(x)), -x))
    order = order[:int((x > -math.inf).sum())]
    if len(order) == 0:
        return [(-1, -math.inf)]
    if t == 0:
        return [(int(order[0]), 0.0)]
    d = 8 * len(x) * 2.0 ** -53
    if 0 < k < len(order):
        order = order[:k]
    y = (x[order] - x[order[0]]) / t
    w = np.exp(y)
    counts = {len(order)}
    if p < 1:
        cum = np.cumsum(w)
        counts = {min(len(order), 1 + int(np.searchsorted(cum, max(p, 0.0) * cum[-1] * (1 + e), side="left"))) for e in (-d, 0, d)}
    if least > 0:
        at = math.log(min(least, 1.0))
        allowed = {int((y >= at * (1 + e)).sum()) for e in (-4 * 2.0 ** -53, 0, 4 * 2.0 ** -53)}
        counts = {max(1, min(a, b)) for a in counts for b in allowed}
    found = {}
    for n in counts:
        by_column = np.argsort(order[:n])
        cum = np.cumsum(w[:n][by_column])
        for e in (-d, 0, d):
            at = int(np.searchsorted(cum, min(u, 1.0) * cum[-1] * (1 + e), side="right"))
            at = min(at, int(np.flatnonzero(w[:n][by_column] > 0)[-1]))
            i = by_column[at]
            found[(int(order[i]), n)] = float(y[i] - math.log(cum[-1]))
    return [(i, lp) for (i, _), lp in found.items()]


def logprob_bound(lp, vocab):
    """ln of a sum of 32-bit weights, each off by 2 ln(vocab) + 4 steps of 2^-24 at most on average, added in 16 steps; one rounding."""
    return (2 * math.log(vocab) + 20) * U + abs(lp) * U + 1e-12


class Limits:
    """Random numbers and limits of n rows; None for an array that is not given."""

    def __init__(self, seed, n, temperature=None, top_k=None, top_p=None, min_p=None, mixed=False, uniform=None):
        rng = np.random.default_rng(seed)
        self.u = rng.random(n) if uniform is None else np.asarray(uniform, np.float64)

        def rows_of(value, dtype, off, spread):
            if value is None:
                return None
            a = np.full(n, value, np.float64)
            if mixed:
                a = spread(a, rng.random(n))
                a[rng.random(n) < 0.25] = off
            return a.astype(dtype)

        self.t = rows_of(temperature, np.float32, 1.0, lambda a, r: a * (0.5 + r))
        if mixed and self.t is not None:
            self.t[rng.random(n) < 0.1] = 0.0
        self.k = rows_of(top_k, np.int32, 0, lambda a, r: np.maximum(1, a * (0.3 + 1.4 * r)))
        self.p = rows_of(top_p, np.float32, 1.0, lambda a, r: a * (0.3 + 0.7 * r))
        self.m = rows_of(min_p, np.float32, 0.0, lambda a, r: a * (0.3 + r))
        if mixed:
            self.u[rng.random(n) < 0.1] = -1.0

    def row(self, r):
        return (float(self.t[r]) if self.t is not None else 1.0, int(self.k[r]) if self.k is not None else 0,
                float(self.p[r]) if self.p is not None else 1.0, float(self.m[r]) if self.m is not None else 0.0, float(self.u[r]))

    def device(self):
        import torch

        return [None if a is None else torch.from_numpy(a).cuda() for a in (self.u, self.t, self.k, self.p, self.m)]


def ptr(t):
    return 0 if t is None else t.data_ptr()


def draw(tok, x, name, limits, stride=None):
    import torch

    n, vocab = x.shape
    u, t, k, p, m = limits.device()
    ids = torch.full((n + 2,), 77, device="cuda", dtype=torch.int32)
    lp = torch.full((n + 2,), 7.5, device="cuda")
    tok.sample(x.data_ptr(), name, n, vocab, u.data_ptr(), ids[1:].data_ptr(), lp[1:].data_ptr(), ptr(t), ptr(k), ptr(p), ptr(m),
               stride=x.stride(0) if stride is None else stride)
    torch.cuda.synchronize()
    assert ids[0] == 77 and ids[-1] == 77 and lp[0] == 7.5 and lp[-1] == 7.5
    return ids[1:-1].cpu().numpy(), lp[1:-1].cpu().numpy()


def check_draws(x, limits, ids, lp, only=None):
    x = x.double().cpu().numpy()
    for r in range(len(ids)) if only is None else only:
        may = possible_draws(x[r if len(x) > 1 else 0], *limits.row(r))
        hit = [want for i, want in may if i == ids[r]]
        assert hit, (r, int(ids[r]), may, limits.row(r))
        if math.isfinite(hit[0]):
            assert any(abs(float(lp[r]) - want) <= logprob_bound(want, x.shape[1]) for want in hit), (r, float(lp[r]), hit, limits.row(r))
        else:
            assert np.array_equal([lp[r]], np.float32([hit[0]]), equal_nan=True), (r, lp[r], hit)


LIMITS = {
    "none": dict(),
    "warm": dict(temperature=1.3),
    "cold": dict(temperature=0.2),
    "greedy": dict(temperature=0.0),
    "k": dict(temperature=0.8, top_k=50),
    "many k": dict(top_k=700),
    "k and p": dict(temperature=0.9, top_k=40, top_p=0.9),
    "many k and p": dict(temperature=1.2, top_k=5000, top_p=0.97),
    "p": dict(temperature=0.7, top_p=0.95),
    "nearly all": dict(temperature=1.1, top_p=0.9999),
    "little p": dict(top_p=0.05),
    "min": dict(min_p=0.05),
    "little min": dict(temperature=1.5, min_p=1e-4),
    "all": dict(temperature=0.9, top_k=100, top_p=0.95, min_p=0.02),
    "mixed": dict(temperature=0.9, top_k=60, top_p=0.95, min_p=0.03, mixed=True),
}
SHAPES = [  # rows, vocabulary, stride, shift
    (1, 50257, 50257, 0),
    (3, 50257, 50304, 1),
    (5, 1000, 1000, 0),
    (4, 777, 777, 3),
    (2, 5, 8, 1),
    (3, 1, 1, 0),
    (2, 131072, 131072, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("which", sorted(LIMITS))
@pytest.mark.parametrize("n,vocab,stride,shift", SHAPES)
def test_sample(tok, name, which, n, vocab, stride, shift):
    x = typed_logits(vocab + n, n, vocab, "text" if vocab >= 1000 else "plain", name, stride, shift)
    limits = Limits(n, n, **LIMITS[which])
    check_draws(x, limits, *draw(tok, x, name, limits))


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("kind", ["plain", "equal", "ties", "zeros", "rising", "falling", "far", "wide", "masked", "lowest", "few", "one"])
@pytest.mark.parametrize("which", ["none", "greedy", "k", "many k", "k and p", "many k and p", "p", "nearly all", "little min", "all"])
def test_sample_of_other_distributions(tok, name, kind, which):
    for n, vocab, stride, shift in ((3, 8193, 8200, 1), (2, 40000, 40000, 0)):
        x = typed_logits(vocab, n, vocab, kind, name, stride, shift)
        limits = Limits(5, n, **LIMITS[which])
        check_draws(x, limits, *draw(tok, x, name, limits))


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("n,vocab", [(200, 3001), (700, 4096), (160, 50257), (2000, 300)])
def test_sample_of_many_rows(tok, name, n, vocab):
    x = typed_logits(n, n, vocab, "text", name)
    for which in ("none", "mixed"):
        limits = Limits(n, n, **LIMITS[which])
        ids, lp = draw(tok, x, name, limits)
        check_draws(x, limits, ids, lp, only=range(0, n, max(1, n * vocab // 2000000)))


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("vocab", [1, 2, 4, 1000, 1024, 40000, 65536])
def test_equal_logits_are_drawn_in_even_parts(tok, name, vocab):
    """Weights of one: sums, shares of them and numbers i / 2^k are exact, and the id at a border is the one behind it."""
    import torch

    n = 64
    u = np.floor(np.random.default_rng(vocab).random(n) * vocab) / vocab if vocab & (vocab - 1) == 0 else np.random.default_rng(vocab).random(n)
    x = torch.zeros(1, vocab, device="cuda", dtype=dtype(name))
    for p in (None, 0.5):
        limits = Limits(1, n, top_p=p, uniform=u)
        kept = vocab if p is None else max(1, (vocab + 1) // 2)  # the fewest of which half the sum is reached
        ids, lp = draw(tok, x.expand(n, vocab), name, limits, stride=0)
        assert np.array_equal(ids, np.floor(u * kept).astype(np.int32))
        assert np.abs(lp + math.log(kept)).max() <= logprob_bound(math.log(kept), vocab)
    limits = Limits(1, n, top_k=max(1, vocab // 4), uniform=u)
    ids, _ = draw(tok, x.expand(n, vocab), name, limits, stride=0)
    assert np.array_equal(ids, np.floor(u * max(1, vocab // 4)).astype(np.int32))


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
def test_more_equal_logits_than_can_be_ranked(tok, name):
    """Limits that fall among a thousand and more equal logits: at the top, and below others."""
    import torch

    x = some_logits(4, 4, 9001, "plain").clamp_(max=0.0).to(dtype(name))   # half of them are zero
    x[1, 77] = x[1, 5000] = 3.0
    x[2] = -7.0
    x[2, ::2] = -math.inf
    x[3, 4000:] = 1.0
    for t, k, p, m in ((1.0, 0, 0.0, 0.0), (1.0, 0, 0.3, 0.0), (1.0, 2000, 1.0, 0.0), (0.7, 2000, 0.4, 0.0), (0.9, 0, 0.99, 0.3), (1.0, 1, 1.0, 0.0)):
        limits = Limits(3, 4, temperature=t, top_k=k, top_p=p, min_p=m)
        check_draws(x, limits, *draw(tok, x, name, limits))


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["none", "k and p", "p", "nearly all", "min", "many k"])
@pytest.mark.parametrize("name", TYPES)
def test_every_column_is_drawn_as_often_as_it_should_be(tok, name, which):
    """One row for all (stride 0) with evenly spaced numbers: column c comes up between S_c n - 1 and S_c n + 1 times, S_c its share."""
    vocab, n = 2000, 4096
    x = typed_logits(5, 1, vocab, "text", name)
    limits = Limits(1, n, **LIMITS[which], uniform=(np.arange(n) + 0.5) / n)
    ids, lp = draw(tok, x.expand(n, vocab), name, limits, stride=0)
    assert (np.diff(ids) >= 0).all()
    got = np.bincount(ids, minlength=vocab)
    for c in np.unique(ids):
        share = math.exp(float(lp[ids == c][0]))
        assert abs(got[c] - share * n) < 1.001
    check_draws(x, limits, ids, lp, only=range(0, n, 17))


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("vocab", [7, 1000, 50257])
def test_sample_at_the_ends(tok, name, vocab):
    """Random numbers at and beyond the ends, limits at theirs, rows without a distribution."""
    import torch

    x = some_logits(3, 1, vocab, "plain").to(dtype(name))
    inf, nan = math.inf, math.nan
    cases = [  # u, temperature, top_k, top_p, min_p
        (0.0, 1, 0, 1, 0), (1.0, 1, 0, 1, 0), (5.0, 1, 0, 1, 0), (inf, 1, 0, 1, 0), (1 - 2.0 ** -53, 1, 0, 1, 0), (2.0 ** -60, 1, 0, 1, 0),
        (0.0, 1, 3, 1, 0), (1.0, 1, 3, 1, 0), (0.0, 1, 0, 0.9, 0), (1.0, 1, 0, 0.9, 0), (0.5, 1, 1, 1, 0), (0.5, 1, -3, 1, 0),
        (0.5, 1, vocab, 1, 0), (0.5, 1, vocab + 5, 1, 0), (0.5, 1, (1 << 31) - 1, 1, 0), (0.5, 1, vocab - 1, 1, 0), (0.5, 1, 0, 0.0, 0),
        (0.5, 1, 0, -1.0, 0), (0.5, 1, 0, 2.0, 0), (0.5, 1, 0, inf, 0), (0.5, 1, 0, -inf, 0), (0.5, 1, 0, 1, 1.0), (0.5, 1, 0, 1, 7.0),
        (0.5, 1, 0, 1, -2.0), (0.5, 1, 0, 1, inf), (0.5, 1, 0, 1, 1e-45), (0.5, 1e-45, 0, 1, 0), (0.5, 1e-30, 5, 0.9, 0), (0.5, 3e38, 0, 1, 0),
        (0.3, 1e30, 0, 0.5, 0), (0.5, 1e-6, 0, 0.9, 0.1), (0.5, 1e6, 7, 0.9, 0.1), (0.5, 0, 0, 1, 0), (-0.0, 1, 0, 1, 0), (-1e-300, 1, 0, 1, 0),
        (-inf, 1, 0, 1, 0), (nan, 1, 0, 1, 0), (0.5, -1, 0, 1, 0), (0.5, inf, 0, 1, 0), (0.5, nan, 0, 1, 0), (0.5, 1, 0, nan, 0),
        (0.5, 1, 0, 1, nan), (-1.0, nan, 0, nan, nan),
    ]
    n = len(cases)
    limits = Limits(1, n)
    limits.u, limits.t, limits.k, limits.p, limits.m = (np.array([c[i] for c in cases], d) for i, d in
                                                        enumerate((np.float64, np.float32, np.int32, np.float32, np.float32)))
    ids, lp = draw(tok, x.expand(n, vocab), name, limits, stride=0)
    check_draws(x, limits, ids, lp)
    # rows that are no distribution
    bad = x.repeat(6, 1)
    bad[0] = -inf
    bad[1, vocab - 1] = nan
    bad[2, 0] = inf
    bad[3] = nan
    bad[4, vocab // 2] = -inf
    bad[5] = inf
    for which in ("none", "greedy", "k and p", "p", "min"):
        limits = Limits(2, 6, **LIMITS[which])
        check_draws(bad, limits, *draw(tok, bad, name, limits))
    limits.u[:] = -1.0
    ids, lp = draw(tok, bad, name, limits)
    assert (ids == -1).all() and (lp == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("t", [1.0, 0.02, 0.01])
@pytest.mark.parametrize("n", [1, 9, 320, 1250])  # eight CTAs to a row or four, one of 256 threads, one of 128
def test_sample_finds_a_nan_wherever_it_lies(tok, name, t, n):
    """A NaN among columns that weigh nothing beside the rest: in sections that are masked otherwise, in front, within and at the end; in
    sections of nothing but NaN; and among logits so far below the highest that a cold temperature leaves nothing of them.  Rows with the
    same masks and no NaN are drawn from."""
    import torch

    vocab = 50257 if n < 100 else 20011
    kinds = 9
    for turn in range(kinds if n < kinds else 1):
        x = some_logits(n + turn, n, vocab, "plain").clamp_(-6.0, 6.0)
        kind = (torch.arange(n, device="cuda") + turn) % kinds
        x[kind == 0, :1024] = -math.inf           # 1024 columns are two sections in 32 bits, one in 16
        x[kind == 0, 700] = math.nan
        x[kind == 1, :1024] = math.nan
        x[kind == 2, :8192] = -math.inf           # the first section of every warp
        x[kind == 2, 8191] = math.nan
        x[kind == 3, vocab - 3000:] = -math.inf
        x[kind == 3, vocab - 1] = math.nan
        x[kind == 4, 0] = math.nan
        x[kind == 4, vocab // 2] = 26.0           # 20 above all others
        x[kind == 5, vocab - 1500] = math.nan
        x[kind == 5, 3] = 26.0
        x[kind == 6, :vocab // 2 + 1] = -math.inf
        x[kind == 6, 5000] = math.nan
        x[kind == 7, :8192] = -math.inf           # no NaN, here and in the last kind
        x[kind == 8, 3] = 26.0
        x = rows(x.to(dtype(name)), name, vocab + 3, 1)
        broken = (kind < 7).cpu().numpy()
        whole = np.flatnonzero(~broken)[:: max(1, n // 40)]
        for which in ("none", "greedy", "k", "many k", "p", "nearly all", "min", "k and p", "all"):
            limits = Limits(n, n, **{**LIMITS[which], **({} if which == "greedy" else {"temperature": t})})
            ids, lp = draw(tok, x, name, limits)
            assert (ids[broken] == -1).all() and np.isnan(lp[broken]).all(), (which, kind[torch.from_numpy(broken).cuda()][:9], ids[broken][:9])
            check_draws(x, limits, ids, lp, only=whole)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_logits_that_32_bits_hardly_hold(tok, name):
    """Logits up to the largest numbers: differences that no 32-bit float holds, and rows of the type's lowest number alone."""
    import torch

    big = float(torch.finfo(dtype(name)).max)
    x = torch.zeros(6, 4001, device="cuda", dtype=dtype(name))
    x[0] = -big
    x[1] = -big
    x[1, 7::9] = big
    x[2, 17] = big
    x[3, ::5] = -big
    x[4] = big
    x[5] = torch.linspace(-3e38, 3e38, 4001, device="cuda").to(x.dtype)
    for which in ("none", "k", "p", "min", "many k and p"):
        limits = Limits(2, 6, **LIMITS[which])
        check_draws(x, limits, *draw(tok, x, name, limits))
    limits = Limits(3, 6, temperature=3e38, top_p=0.7)
    check_draws(x, limits, *draw(tok, x, name, limits))


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("mask", [-1e9, -1e10, -math.inf])
def test_sample_with_whole_ranges_masked(tok, name, mask):
    """Stretches of columns at a number that no other column comes near (-inf here: the type's lowest), at the beginning, within and at the
    end, so that sections and sets of nothing else are looked at."""
    import torch

    low = float(torch.finfo(dtype(name)).min)
    n, vocab = 6, 50257
    x = some_logits(8, n, vocab, "text")
    x[0, 9000:30000] = x[1, :9000] = x[2, 2000:] = x[3, 40000:] = max(mask, low)
    x[4, :16384] = x[4, 16500:] = max(mask, low)
    x[5] = max(mask, low)
    x = rows(x.to(dtype(name)), name, 50304, 1)
    for which in ("none", "greedy", "k", "many k", "many k and p", "p", "nearly all", "little min", "all"):
        limits = Limits(n, n, **LIMITS[which])
        check_draws(x, limits, *draw(tok, x, name, limits))
    limits = Limits(n, n, top_k=45000)       # masked columns are among the first where too few others are there
    check_draws(x, limits, *draw(tok, x, name, limits))


@pytest.mark.gpu
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("mean,deviation", [(10.0, 2.0), (-6.0, 2.0), (18.0, 3.0), (300.0, 2.0)])
def test_sample_of_logits_off_zero(tok, name, mean, deviation):
    """16-bit logits are coarse away from zero: hundreds and thousands of columns are equal at the border of a wide limit."""
    import torch

    x = (torch.randn(3, 131072, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda") * deviation + mean).to(dtype(name))
    for limits in (Limits(1, 3, top_p=0.95), Limits(2, 3, top_k=2000), Limits(3, 3, temperature=0.8, top_k=5000, top_p=0.9), Limits(4, 3),
                   Limits(5, 3, temperature=0.9, top_p=0.9, min_p=1e-3)):
        check_draws(x, limits, *draw(tok, x, name, limits))


@pytest.mark.gpu
def test_sample_without_logprob_and_of_nothing(tok):
    import torch

    x = some_logits(1, 3, 999, "text")
    u = torch.tensor([0.2, 0.9, 0.5], device="cuda", dtype=torch.float64)
    ids, again = (torch.full((3,), 9, device="cuda", dtype=torch.int32) for _ in range(2))
    lp = torch.empty(3, device="cuda")
    tok.sample(x.data_ptr(), "f32", 3, 999, u.data_ptr(), ids.data_ptr())
    tok.sample(x.data_ptr(), "f32", 3, 999, u.data_ptr(), again.data_ptr(), lp.data_ptr())
    assert torch.equal(ids, again)
    tok.sample(0, "f32", 0, 999, 0, 0)
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_largest_vocabulary_and_offsets_beyond_32_bits(tok):
    import torch

    vocab = 1 << 20
    x = typed_logits(9, 2, vocab, "text", "bf16")
    for which in ("none", "k and p", "p", "nearly all"):
        limits = Limits(2, 2, **LIMITS[which])
        check_draws(x, limits, *draw(tok, x, "bf16", limits))
    stride = (1 << 31) + 8
    whole = torch.empty(2 * stride + 1000, device="cuda", dtype=torch.bfloat16)
    view = whole.as_strided((3, 1000), (stride, 1))
    view.copy_(some_logits(4, 3, 1000, "text"))
    limits = Limits(3, 3, **LIMITS["k and p"])
    check_draws(view, limits, *draw(tok, view, "bf16", limits))


@pytest.mark.gpu
def test_the_same_draws_every_time(tok):
    for name, n, vocab in (("bf16", 300, 50257), ("f32", 7, 131072), ("f16", 40, 3001)):
        x = typed_logits(n, n, vocab, "text", name)
        limits = Limits(n, n, **LIMITS["mixed"])
        ids, lp = draw(tok, x, name, limits)
        for _ in range(5):
            i2, l2 = draw(tok, x, name, limits)
            assert np.array_equal(ids, i2) and np.array_equal(lp, l2, equal_nan=True)


# ---------------------------------------------------------------------------------------------------- blocks and slots
class Pool:
    """Requests with their blocks, and the ring of free ones, on the host as the definition has it."""

    def __init__(self, seed, n, block, columns, stride, blocks, head=0, old=None):
        rng = np.random.default_rng(seed)
        self.n, self.block, self.columns, self.stride = n, block, columns, stride
        self.old = (np.exp(rng.random(n) * math.log(columns * block + 1.0)) - 1).astype(np.int64) if old is None else np.asarray(old)
        held = -(-np.maximum(self.old, 0) // block)
        ids = rng.permutation(blocks).astype(np.int32)
        used = int(held.sum())
        assert used <= blocks
        self.table = np.full((n, stride), -7, np.int32)
        at = 0
        for r in range(n):
            self.table[r, :held[r]] = ids[at:at + held[r]]
            at += held[r]
        self.queue = np.full(blocks, -9, np.int32)
        self.queue[(head + np.arange(blocks - used)) % blocks] = ids[used:]
        self.head, self.tail = head, head + blocks - used

    def step(self, new):
        """Returns the status; applies the step where it is 0."""
        both = (self.old >= 0) & (new >= 0)
        have, need = (np.where(both, -(-a // self.block), 0) for a in (self.old, new))
        took, gave = int(np.maximum(need - have, 0).sum()), int(np.maximum(have - need, 0).sum())
        size = len(self.queue)
        if max(have.max(initial=0), need.max(initial=0)) > self.columns:
            return -1
        if self.tail < self.head or self.tail - self.head + gave > size:
            return -2
        if took > self.tail - self.head:
            return took - (self.tail - self.head)
        for r in range(self.n):
            for c in range(have[r], need[r]):
                self.table[r, c] = self.queue[self.head % size]
                self.head += 1
        for r in range(self.n):
            for c in range(need[r], have[r]):
                self.queue[self.tail % size] = self.table[r, c]
                self.tail += 1
        self.old = np.where(both, new, self.old)
        return 0


def run_tables(tok, pool, new, in_place=False):
    """The step on the GPU from the pool's present state: (table, queue, state_out)."""
    import torch

    old, new = (torch.from_numpy(np.asarray(a, np.int32)).cuda() for a in (pool.old, new))
    table = torch.from_numpy(pool.table.copy()).cuda()
    queue = torch.from_numpy(pool.queue.copy()).cuda()
    state = torch.tensor([pool.head, pool.tail, 55], dtype=torch.int64, device="cuda")
    out = state if in_place else torch.full((3,), 66, dtype=torch.int64, device="cuda")
    tok.block_tables(old.data_ptr(), new.data_ptr(), pool.n, pool.block, table.data_ptr(), pool.columns, queue.data_ptr(), len(pool.queue),
                     state.data_ptr(), out.data_ptr(), table_stride=pool.stride)
    torch.cuda.synchronize()
    if not in_place:
        assert state.tolist() == [pool.head, pool.tail, 55]
    return table.cpu().numpy(), queue.cpu().numpy(), out.cpu().tolist()


def check_step(tok, pool, new, in_place=False):
    got = run_tables(tok, pool, new, in_place)
    status = pool.step(np.asarray(new))
    assert got[2] == [pool.head, pool.tail, status]
    assert np.array_equal(got[0], pool.table) and np.array_equal(got[1], pool.queue)
    return status


def slots_of(tok, pool, old, new, capacity, state=None, wanted=("positions", "requests")):
    import torch

    old, new = (torch.from_numpy(np.asarray(a, np.int32)).cuda() for a in (old, new))
    table = torch.from_numpy(pool.table).cuda()
    slots, offsets = (torch.full((k + 2,), 77, dtype=torch.int64, device="cuda") for k in (capacity, pool.n + 1))
    positions, requests = (torch.full((capacity + 2,), 77, dtype=torch.int32, device="cuda") for _ in range(2))
    d_state = None if state is None else torch.tensor(state, dtype=torch.int64, device="cuda")
    tok.slot_map(old.data_ptr(), new.data_ptr(), pool.n, pool.block, table.data_ptr(), pool.columns, capacity, slots[1:].data_ptr(),
                 offsets[1:].data_ptr(), positions[1:].data_ptr() if "positions" in wanted else 0,
                 requests[1:].data_ptr() if "requests" in wanted else 0, ptr(d_state), table_stride=pool.stride)
    torch.cuda.synchronize()
    out = [a.cpu().numpy() for a in (slots, positions, requests, offsets)]
    assert all(a[0] == 77 and a[-1] == 77 for a in out)
    return [a[1:-1] for a in out]


def want_slots(pool, old, new, capacity, done=True):
    old, new = np.asarray(old, np.int64), np.asarray(new, np.int64)
    more = np.where((old >= 0) & (new > old) & done, new - old, 0)
    offsets = np.concatenate([[0], np.cumsum(more)])
    r = np.repeat(np.arange(pool.n), more)
    j = old[r] + np.arange(len(r)) - offsets[r]
    column = j // pool.block
    entry = np.where(column < pool.columns, pool.table[r, np.minimum(column, pool.columns - 1)].astype(np.int64), -1)
    slot = np.where(entry >= 0, entry * pool.block + j % pool.block, -1)
    full = [np.full(capacity, -1, np.int64) for _ in range(3)]
    k = min(capacity, len(r))
    full[0][:k], full[1][:k], full[2][:k] = slot[:k], j[:k], r[:k]
    return full + [offsets]


def check_slots(tok, pool, old, new, capacity, state=None):
    got = slots_of(tok, pool, old, new, capacity, state)
    for g, w in zip(got, want_slots(pool, old, new, capacity, state is None or state[2] == 0)):
        assert np.array_equal(g, w)


def next_lengths(seed, old, longest, kind):
    rng = np.random.default_rng(seed)
    n = len(old)
    new = np.minimum(old + 1, longest)
    if kind == "replace":
        new = np.where(rng.random(n) < 0.5, new, (np.exp(rng.random(n) * math.log(longest + 1.0)) - 1).astype(np.int64))
    if kind in ("step", "replace"):
        new[rng.random(n) < 0.1] = 0
    if kind == "gone":
        new[:] = 0
    if kind == "full":
        new[:] = longest
    if kind == "negative":
        new[rng.random(n) < 0.3] = -1
        new[rng.random(n) < 0.1] = -(1 << 31)
    return new


POOLS = [  # requests, tokens a block, columns, stride
    (1, 16, 8, 8), (1, 1, 1, 1), (3, 1, 50, 64), (2, 128, 1, 1), (33, 24, 20, 21), (257, 16, 40, 40), (1000, 7, 9, 16), (1024, 16, 3, 3),
    (1025, 64, 30, 32), (5000, 16, 12, 12), (20000, 32, 5, 5), (3, 16, 5000, 5000), (2, 1000, 300, 300),
]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["one more", "step", "replace", "gone", "full", "negative"])
@pytest.mark.parametrize("n,block,columns,stride", POOLS)
def test_block_tables_and_slots(tok, n, block, columns, stride, kind):
    blocks = n * columns + 5
    pool = Pool(n, n, block, columns, stride, blocks, head=blocks * 1000 + 3)
    if kind == "negative":
        pool.old[::3] = -1
    old = pool.old.copy()
    new = next_lengths(n, old, columns * block, kind)
    assert check_step(tok, pool, new) == 0
    total = int(np.where((old >= 0) & (new > old), new - old, 0).sum())
    for capacity in {min(total, 1 << 20), min(total, 1 << 20) + 37, max(0, min(total, 1 << 20) - 5), 0}:
        check_slots(tok, pool, old, new, capacity)
    assert check_step(tok, pool, next_lengths(n + 1, np.maximum(pool.old, 0), columns * block, "replace"), in_place=True) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("n", [152000, 200001])
def test_more_requests_than_ctas_have_threads(tok, n):
    """More than 1024 requests to each CTA of any GPU's: tiles behind the first go on where it has ended."""
    pool = Pool(n, n, 16, 2, 2, 2 * n + 5, head=77)
    for i, kind in enumerate(("replace", "full", "step", "gone")):
        old = pool.old.copy()
        new = next_lengths(i, old, 32, kind)
        assert check_step(tok, pool, new, in_place=i % 2 == 1) == 0
        total = int(np.where(new > old, new - old, 0).sum())
        check_slots(tok, pool, old, new, min(total, 1 << 20) + 5)


@pytest.mark.gpu
@pytest.mark.parametrize("n,every", [(20000, 10), (20000, 9999), (100000, 100), (8193, 8193)])
def test_slots_of_few_among_many_requests(tok, n, every):
    """Few of many requests have new tokens: those of a CTA lie among more requests than its shared memory has room for."""
    pool = Pool(n, n, 16, 3, 3, 3 * n)
    new = pool.old.copy()
    new[every // 2::every] = np.minimum(new[every // 2::every] + 1, 48)
    new[every // 3::every] = np.maximum(new[every // 3::every] - 1, 0)
    total = int(np.where(new > pool.old, new - pool.old, 0).sum())
    far = pool.old.copy()
    far[[0, n - 1]] += 700
    assert check_step(tok, Pool(n, n, 16, 3, 3, 3 * n, old=pool.old), new) == 0
    for capacity in (total, total + 3000, max(1, total // 2)):
        check_slots(tok, pool, pool.old, new, capacity)
    check_slots(tok, pool, pool.old, far, 1500)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 50, 1024, 3000])
def test_steps_that_are_not_done(tok, n):
    block, columns = 16, 20
    tight = Pool(n, n, block, columns, columns + 1, n * columns, head=0)
    more = np.minimum(tight.old + 300, columns * block)
    wanted = int((-(-more // block) - -(-tight.old // block)).sum())
    tight.tail = tight.head + wanted - 1                        # one block too few
    before = [tight.table.copy(), tight.queue.copy()]
    if wanted:
        assert check_step(tok, tight, more) == 1
        assert check_step(tok, tight, more, in_place=True) == 1
        check_slots(tok, tight, tight.old, more, 100, state=[tight.head, tight.tail, 1])
        check_slots(tok, tight, tight.old, more, 100, state=[tight.head, tight.tail, -2])
        check_slots(tok, tight, tight.old, more, 100, state=[tight.head, tight.tail, 0])
        tight.tail += 1                                         # just enough
        assert check_step(tok, tight, more) == 0
    beyond = Pool(n, n, block, columns, columns, n * columns + n + 8)
    new = beyond.old.copy()
    new[n // 2] = columns * block + 1
    assert check_step(tok, beyond, new) == -1
    new[n // 2] = (1 << 31) - 1
    assert check_step(tok, beyond, new) == -1
    broken = Pool(n, n, block, columns, columns, n * columns)
    broken.old[:] = 17                                          # the ring is too full for what comes back
    broken.tail = broken.head + len(broken.queue) - 1
    assert check_step(tok, broken, np.zeros(n, np.int64)) == -2
    broken.tail = broken.head - 1
    assert check_step(tok, broken, broken.old) == -2
    broken.tail = broken.head + len(broken.queue) + 1
    assert check_step(tok, broken, broken.old) == -2
    assert before[1].shape == tight.queue.shape


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 50, 512, 3000])
@pytest.mark.parametrize("in_place", [False, True])
def test_steps_with_queues_that_cannot_be(tok, n, in_place):
    """Counts at the ends of 64 bits, whose differences and sums pass them; a full queue that gets blocks back though as many are taken."""
    most, least, block, columns = (1 << 63) - 1, -(1 << 63), 16, 4
    pool = Pool(n, n, block, columns, columns, n * columns, old=np.full(n, 33))  # three blocks each
    size = len(pool.queue)
    back = np.full(n, 33)
    back[n // 2] = 0
    both = back.copy()
    both[-1] = 64 if n > 1 else 0
    for head, tail in ((0, most), (1, least), (0, least), (least, most), (least, least), (-1, 5), (-5, -1), (most, 0), (most, least), (5, 4),
                       (most - 1, most), (most, most), (most - 2, most - 2), (0, size + 1), (most - size - 1, most), (7, 7 + size)):
        pool.head, pool.tail = head, tail
        for new in (back, both):
            table, queue, state = run_tables(tok, pool, new, in_place)
            assert state == [head, tail, -2], (head, tail)
            assert np.array_equal(table, pool.table) and np.array_equal(queue, pool.queue)
    # the last counts that there are
    pool.head, pool.tail = most - 4, most - 3
    assert check_step(tok, pool, back, in_place) == 0 and (pool.head, pool.tail) == (most - 4, most)
    grown = pool.old.copy()
    grown[0] += 16
    if n > 1:
        assert check_step(tok, pool, grown, in_place) == 0 and pool.head == most - 3


@pytest.mark.gpu
def test_steps_of_no_requests(tok):
    import torch

    state = torch.tensor([3, 9, 4], dtype=torch.int64, device="cuda")
    out = torch.zeros(3, dtype=torch.int64, device="cuda")
    queue = torch.zeros(10, dtype=torch.int32, device="cuda")
    tok.block_tables(0, 0, 0, 16, 0, 4, queue.data_ptr(), 10, state.data_ptr(), out.data_ptr())
    assert out.tolist() == [3, 9, 0]
    offsets, slots = torch.full((1,), 5, dtype=torch.int64, device="cuda"), torch.full((7,), 5, dtype=torch.int64, device="cuda")
    tok.slot_map(0, 0, 0, 16, 0, 4, 7, slots.data_ptr(), offsets.data_ptr())
    assert offsets.tolist() == [0] and slots.tolist() == [-1] * 7
    tok.slot_map(0, 0, 0, 16, 0, 4, 0, 0, offsets.data_ptr())
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("wanted", [(), ("positions",), ("requests",)])
def test_slots_alone(tok, wanted):
    pool = Pool(3, 40, 16, 9, 9, 400)
    new = np.minimum(pool.old + 5, 144)
    pool.table[:, 4] = -3                                       # entries that are no blocks give no slots
    got = slots_of(tok, pool, pool.old, new, 210, wanted=wanted)
    want = want_slots(pool, pool.old, new, 210)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[3], want[3])
    for name, g, w in (("positions", got[1], want[1]), ("requests", got[2], want[2])):
        assert np.array_equal(g, w) if name in wanted else (g == 77).all()


@pytest.mark.gpu
def test_slots_beyond_32_bits(tok):
    """Blocks whose first slot is beyond 2^31, a table whose rows are, and positions up to the last."""
    import torch

    block, columns, stride = 1 << 20, 2047, (1 << 30) + 5
    table = torch.empty(2 * stride + columns, dtype=torch.int32, device="cuda")
    view = table.as_strided((3, columns), (stride, 1))
    view.copy_(torch.arange(3 * columns, device="cuda").view(3, columns) + (1 << 20))
    last = (1 << 31) - 1
    old = torch.tensor([5 * block - 2, last - 3, 0], dtype=torch.int32, device="cuda")
    new = torch.tensor([5 * block + 2, last, 3], dtype=torch.int32, device="cuda")
    slots, offsets = torch.empty(12, dtype=torch.int64, device="cuda"), torch.empty(4, dtype=torch.int64, device="cuda")
    positions = torch.empty(12, dtype=torch.int32, device="cuda")
    tok.slot_map(old.data_ptr(), new.data_ptr(), 3, block, table.data_ptr(), columns, 12, slots.data_ptr(), offsets.data_ptr(),
                 positions.data_ptr(), table_stride=stride)
    assert offsets.tolist() == [0, 4, 7, 10]
    j = [5 * block - 2 + i for i in range(4)] + [last - 3 + i for i in range(3)] + [0, 1, 2]
    r = [0] * 4 + [1] * 3 + [2] * 3
    want = [(r[i] * columns + j[i] // block + (1 << 20)) * block + j[i] % block if j[i] // block < columns else -1 for i in range(10)]
    assert slots.tolist() == want + [-1, -1] and positions.tolist() == j + [-1, -1]


# ---------------------------------------------------------------------------------------------------- together
@pytest.mark.gpu
def test_generation_from_text(native_built, merges_path):
    """Prompts are tokenised on the GPU, get blocks and slots, and grow by drawn ids for some steps: each request reads its own
    tokens back through its blocks, and in the end all blocks are in the queue again."""
    import torch

    import gputok_b200

    t = Tokenizer(merges_path, 1 << 16, 50, device=0)
    t.set_stream(torch.cuda.current_stream().cuda_stream)
    n, vocab, dim, block, columns, steps = 9, 50257, 32, 16, 40, 6
    texts = [gputok_b200.TextGen(i).text(200 + 90 * i).tobytes() for i in range(n)]
    d_bytes = torch.from_numpy(np.frombuffer(b"".join(texts), np.uint8).copy()).cuda()
    d_off = torch.tensor(np.cumsum([0] + [len(x) for x in texts]), dtype=torch.int64, device="cuda")
    ids = torch.empty(len(d_bytes), dtype=torch.int32, device="cuda")
    chunk_off = torch.empty(n + 1, dtype=torch.int64, device="cuda")
    total, chunks, _ = t.encode_device(d_bytes.data_ptr(), len(d_bytes), d_off.data_ptr(), n, ids.data_ptr(), len(d_bytes),
                                       chunk_off.data_ptr(), n + 1)
    assert chunks == n
    blocks = n * columns
    table = torch.full((n, columns), -1, dtype=torch.int32, device="cuda")
    queue = torch.randperm(blocks, device="cuda").to(torch.int32)
    everything = queue.clone()
    state = torch.tensor([0, blocks, 0], dtype=torch.int64, device="cuda")
    cache = torch.full((blocks * block, dim), math.nan, device="cuda")
    embedding = torch.randn(vocab, dim, device="cuda")
    old = torch.zeros(n, dtype=torch.int32, device="cuda")
    new = chunk_off.diff().to(torch.int32)
    texts_so_far = [ids[int(chunk_off[r]):int(chunk_off[r + 1])].tolist() for r in range(n)]
    tokens = ids[:total].contiguous()
    g = torch.Generator(device="cuda").manual_seed(1)
    for step in range(steps):
        capacity = len(tokens) + 3
        slots = torch.empty(capacity, dtype=torch.int64, device="cuda")
        positions, requests = (torch.empty(capacity, dtype=torch.int32, device="cuda") for _ in range(2))
        offsets = torch.empty(n + 1, dtype=torch.int64, device="cuda")
        t.block_tables(old.data_ptr(), new.data_ptr(), n, block, table.data_ptr(), columns, queue.data_ptr(), blocks, state.data_ptr(),
                       state.data_ptr())
        t.slot_map(old.data_ptr(), new.data_ptr(), n, block, table.data_ptr(), columns, capacity, slots.data_ptr(), offsets.data_ptr(),
                   positions.data_ptr(), requests.data_ptr(), state.data_ptr())
        x = torch.empty(len(tokens), dim, device="cuda")
        t.embed(tokens.data_ptr(), len(tokens), embedding.data_ptr(), "f32", vocab, dim, x.data_ptr(), "f32")
        assert state[2] == 0 and int(offsets[-1]) == len(tokens) and (slots[-3:] == -1).all()
        cache[slots[:-3]] = x
        # a stand-in for the model: the mean of what a request's blocks hold, against the table
        means = []
        for r in range(n):
            length = int(new[r])
            j = torch.arange(length, device="cuda")
            mine = cache[table[r].long()[j // block] * block + j % block]
            assert torch.equal(mine, embedding[torch.tensor(texts_so_far[r], device="cuda")])
            means.append(mine.mean(0))
        logits = (torch.stack(means) @ embedding.T * 3).to(torch.bfloat16)
        limits = Limits(step, n, temperature=0.8, top_k=50, top_p=0.9)
        u, temp, k, p, _ = limits.device()
        drawn = torch.empty(n, dtype=torch.int32, device="cuda")
        lp, check = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
        t.sample(logits.data_ptr(), "bf16", n, vocab, u.data_ptr(), drawn.data_ptr(), lp.data_ptr(), temp.data_ptr(), k.data_ptr(), p.data_ptr())
        t.token_logprobs(logits.data_ptr(), "bf16", n, vocab, drawn.data_ptr(), check.data_ptr(), scale=1 / 0.8)
        check_draws(logits, limits, drawn.cpu().numpy(), lp.cpu().numpy())
        assert (check <= lp + 1e-4).all()         # fewer ids share the probability
        for r in range(n):
            texts_so_far[r].append(int(drawn[r]))
        tokens = drawn
        old, new = new, new + 1
    t.block_tables(old.data_ptr(), torch.zeros_like(old).data_ptr(), n, block, table.data_ptr(), columns, queue.data_ptr(), blocks,
                   state.data_ptr(), state.data_ptr())
    head, tail, status = state.tolist()
    assert status == 0 and tail - head == blocks
    assert torch.equal(queue.sort().values, everything.sort().values)
    assert len(t.decode(texts_so_far[0])) > 200
    del g


@pytest.mark.gpu
def test_a_step_captured_and_replayed(native_built, merges_path):
    """Blocks, slots and ids of a step in one graph, whose lengths and states move on in place; the handle's first calls."""
    import torch

    t = Tokenizer(merges_path, 2048, 50, device=0)
    n, vocab, block, columns = 70, 3001, 16, 12
    pool = Pool(3, n, block, columns, columns, n * columns, old=np.arange(n) * 2)
    old, new = (torch.from_numpy(a.astype(np.int32)).cuda() for a in (pool.old, pool.old + 1))
    table, queue = torch.from_numpy(pool.table.copy()).cuda(), torch.from_numpy(pool.queue.copy()).cuda()
    state = torch.tensor([pool.head, pool.tail, 0], dtype=torch.int64, device="cuda")
    slots, offsets = torch.empty(n, dtype=torch.int64, device="cuda"), torch.empty(n + 1, dtype=torch.int64, device="cuda")
    x = typed_logits(1, n, vocab, "text", "bf16")
    limits = Limits(1, n, **LIMITS["mixed"])
    u, temp, k, p, m = limits.device()
    ids, lp = torch.empty(n, dtype=torch.int32, device="cuda"), torch.empty(n, device="cuda")
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    t.set_stream(s.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        t.block_tables(old.data_ptr(), new.data_ptr(), n, block, table.data_ptr(), columns, queue.data_ptr(), len(pool.queue),
                       state.data_ptr(), state.data_ptr())
        t.slot_map(old.data_ptr(), new.data_ptr(), n, block, table.data_ptr(), columns, n, slots.data_ptr(), offsets.data_ptr(),
                   d_state=state.data_ptr())
        t.sample(x.data_ptr(), "bf16", n, vocab, u.data_ptr(), ids.data_ptr(), lp.data_ptr(), temp.data_ptr(), k.data_ptr(), p.data_ptr(),
                 m.data_ptr())
        old.copy_(new)
        new.add_(1)
    for step in range(20):
        x.copy_(some_logits(step + 5, n, vocab, "text"))
        now = pool.old.copy()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert pool.step(now + 1) == 0
        assert state.tolist() == [pool.head, pool.tail, 0]
        assert np.array_equal(table.cpu().numpy(), pool.table) and np.array_equal(queue.cpu().numpy(), pool.queue)
        assert np.array_equal(slots.cpu().numpy(), want_slots(pool, now, now + 1, n)[0])
        check_draws(x, limits, ids.cpu().numpy(), lp.cpu().numpy(), only=range(step % 7, n, 7))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [600, 9000])
def test_steps_of_many_requests_captured_and_replayed(native_built, merges_path, n):
    """Calls of two kernels each, in one graph behind each other and behind what moves their lengths on."""
    import torch

    t = Tokenizer(merges_path, 2048, 50, device=0)
    block, columns, vocab = 4, 6, 300
    pool = Pool(5, n, block, columns, columns, n * columns, old=np.arange(n) % 3)
    old, new = (torch.from_numpy(a.astype(np.int32)).cuda() for a in (pool.old, pool.old + 1))
    table, queue = torch.from_numpy(pool.table.copy()).cuda(), torch.from_numpy(pool.queue.copy()).cuda()
    state = torch.tensor([pool.head, pool.tail, 0], dtype=torch.int64, device="cuda")
    capacity = 5 * n
    slots, offsets = (torch.empty(k, dtype=torch.int64, device="cuda") for k in (capacity, n + 1))
    positions, requests = (torch.empty(capacity, dtype=torch.int32, device="cuda") for _ in range(2))
    x = typed_logits(1, n, vocab, "text", "bf16")
    limits = Limits(1, n, **LIMITS["mixed"])
    u, temp, k, p, m = limits.device()
    ids, lp = torch.empty(n, dtype=torch.int32, device="cuda"), torch.empty(n, device="cuda")
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    t.set_stream(s.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        t.block_tables(old.data_ptr(), new.data_ptr(), n, block, table.data_ptr(), columns, queue.data_ptr(), len(pool.queue),
                       state.data_ptr(), state.data_ptr())
        t.slot_map(old.data_ptr(), new.data_ptr(), n, block, table.data_ptr(), columns, capacity, slots.data_ptr(), offsets.data_ptr(),
                   positions.data_ptr(), requests.data_ptr(), state.data_ptr())
        t.sample(x.data_ptr(), "bf16", n, vocab, u.data_ptr(), ids.data_ptr(), lp.data_ptr(), temp.data_ptr(), k.data_ptr(), p.data_ptr(),
                 m.data_ptr())
        old.copy_(new)
        new.add_(torch.where(new % 7 == 3, 5, 1)).remainder_(columns * block)  # some bring several, some end
    for step in range(12):
        x.copy_(some_logits(step + 5, n, vocab, "text"))
        now, then = pool.old.copy(), new.cpu().numpy().astype(np.int64)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert pool.step(then) == 0
        assert state.tolist() == [pool.head, pool.tail, 0]
        assert np.array_equal(table.cpu().numpy(), pool.table) and np.array_equal(queue.cpu().numpy(), pool.queue)
        for got, want in zip((slots, positions, requests, offsets), want_slots(pool, now, then, capacity)):
            assert np.array_equal(got.cpu().numpy(), want)
        check_draws(x, limits, ids.cpu().numpy(), lp.cpu().numpy(), only=range(step, n, 61))


@pytest.mark.gpu
def test_two_handles_on_two_streams(native_built, merges_path):
    """Calls of two handles at once give what they give alone."""
    import torch

    handles = [Tokenizer(merges_path, 2048, 50, device=0) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    sets = []
    for i, t in enumerate(handles):
        t.set_stream(streams[i].cuda_stream)
        n, vocab = (60, 50257) if i else (200, 9001)
        x = typed_logits(i, n, vocab, "text", "bf16")
        limits = Limits(i, n, **LIMITS["mixed"])
        pool = Pool(i, 900, 16, 30, 30, 900 * 30)
        new = next_lengths(i, pool.old, 480, "replace")
        out = [torch.empty(n, dtype=torch.int32, device="cuda"), torch.empty(n, device="cuda")]
        arrays = [torch.from_numpy(a).cuda() for a in (pool.old.astype(np.int32), new.astype(np.int32), pool.table, pool.queue)]
        arrays += [torch.tensor([pool.head, pool.tail, 0], dtype=torch.int64, device="cuda"), torch.empty(3, dtype=torch.int64, device="cuda")]
        slots, offsets = torch.empty(200000, dtype=torch.int64, device="cuda"), torch.empty(901, dtype=torch.int64, device="cuda")
        sets.append((t, x, n, vocab, limits, limits.device(), out, pool, new, arrays, slots, offsets))
    torch.cuda.synchronize()
    for _ in range(20):
        for t, x, n, vocab, limits, dev, out, pool, new, arr, slots, offsets in sets:
            u, temp, k, p, m = dev
            t.sample(x.data_ptr(), "bf16", n, vocab, u.data_ptr(), out[0].data_ptr(), out[1].data_ptr(), temp.data_ptr(), k.data_ptr(),
                     p.data_ptr(), m.data_ptr())
            t.block_tables(arr[0].data_ptr(), arr[1].data_ptr(), 900, 16, arr[2].data_ptr(), 30, arr[3].data_ptr(), len(pool.queue),
                           arr[4].data_ptr(), arr[5].data_ptr())
            t.slot_map(arr[0].data_ptr(), arr[1].data_ptr(), 900, 16, arr[2].data_ptr(), 30, 200000, slots.data_ptr(), offsets.data_ptr(),
                       d_state=arr[5].data_ptr())
    torch.cuda.synchronize()
    for t, x, n, vocab, limits, dev, out, pool, new, arr, slots, offsets in sets:
        check_draws(x, limits, out[0].cpu().numpy(), out[1].cpu().numpy(), only=range(0, n, 5))
        now = pool.old.copy()
        assert pool.step(new) == 0
        assert np.array_equal(arr[2].cpu().numpy(), pool.table) and arr[5].tolist() == [pool.head, pool.tail, 0]
        assert np.array_equal(slots.cpu().numpy(), want_slots(pool, now, new, 200000)[0])


@pytest.mark.gpu
def test_checked_build_of_a_step(native_built):
    """The library with index checks (-DGTK_CHECKED) through cases of this file, in a process of its own: no check of an index may
    fail.  Before that a check in either source file is made to fail, and is reported with its number, value and limit."""
    import os
    import subprocess
    import sys

    from gputok_b200.capi import checked_library_path

    path = checked_library_path()
    probe = ("import ctypes,sys; lib=ctypes.CDLL(sys.argv[1]); w=(ctypes.c_int*4)()\n"
             "for t in (4, 5, 0): print(lib.gtk_debug_check_words(w, 1, t), *w)")
    out = subprocess.run([sys.executable, "-c", probe, path], capture_output=True, text=True, timeout=300)
    assert out.stdout.split("\n")[:3] == ["0 499 5 4 1", "0 599 5 4 1", "0 0 0 0 0"], out.stdout + out.stderr
    chosen = "(test_sample or equal_logits or every_column or hardly_hold or test_block or not_done or generation or captured) and not checked"
    run = subprocess.run([sys.executable, "-m", "pytest", os.path.abspath(__file__), "-m", "gpu", "-x", "-q", "-s", "-k", chosen],
                         capture_output=True, text=True, timeout=1500, env=dict(os.environ, GPUTOK_B200_LIBRARY=path))
    assert run.returncode == 0, run.stdout[-3000:] + run.stderr[-2000:]
    assert "CHECKED_BUILD rc=0 failures=0" in run.stdout, run.stdout[-2000:]
