"""Picks under top-k, top-p and min-p against the plain form in 64 bits."""
import numpy as np
import pytest
import torch

import plain_continuations as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def ops():
    from imparo_amd.kernels import ops as o
    return o


def run(x, temperature, u, top_k=None, top_p=None, min_p=None):
    n = x.shape[0]
    to = lambda a, t: None if a is None else torch.tensor(np.asarray(a), dtype=t, device=DEV)
    out = torch.full((n,), -7, dtype=torch.int32, device=DEV)
    back = ops().sample_rows(torch.from_numpy(x).to(DEV), to(temperature, torch.float32), to(u, torch.float32), out,
                             top_k=to(top_k, torch.int32), top_p=to(top_p, torch.float32), min_p=to(min_p, torch.float32))
    assert back is out
    return out.cpu().tolist()


def check(x, temperature, u, top_k, top_p, min_p):
    got = run(x, temperature, u, top_k, top_p, min_p)
    f32 = lambda a: [float(np.float32(v)) for v in a]
    want = [plain.pick(x[r], f32(temperature)[r], f32(u)[r], top_k[r], f32(top_p)[r], f32(min_p)[r]) for r in range(len(got))]
    assert got == want, [(r, g, w) for r, (g, w) in enumerate(zip(got, want)) if g != w]


def filters_of(rng, n, vocab):
    """Every row some filter, the awkward values among them."""
    top_k = rng.choice([0, 1, 2, 7, 50, max(1, vocab - 1)], n)
    top_p = rng.choice([1.0, 0.999, 0.9, 0.5, 1e-6], n)
    min_p = rng.choice([0.0, 0.001, 0.05, 0.5, 1.0], n)
    top_p = np.where((top_k == 0) & (min_p == 0) & (top_p == 1.0), 0.95, top_p)
    return top_k.tolist(), top_p.tolist(), min_p.tolist()


@pytest.mark.parametrize("vocab", [2, 5, 63, 1003, 4097, 16383, 16384, 50257, 65536, 130001])
@pytest.mark.parametrize("values", ["normal", "steep", "flat", "quarters", "gaps"])
def test_picks(vocab, values):
    rng = np.random.default_rng(vocab)
    n = 24 if vocab < 20000 else 12
    x = rng.standard_normal((n, vocab)).astype(np.float32) * {"steep": 20.0, "flat": 0.1}.get(values, 2.0)
    if values == "quarters":
        x = np.round(x * 4) / 4                                   # many ties
    if values == "gaps":
        x[:, ::3] = np.nan
        x[::2, 1::4] = -np.inf
        x[:, -1] = 1.5
    u = rng.integers(0, 1 << 24, n) / float(1 << 24)
    u[0], u[1], u[2] = 0.0, 1 - 2.0 ** -24, 1.0
    check(x.astype(np.float32), rng.uniform(0.3, 1.5, n), u, *filters_of(rng, n, vocab))


@pytest.mark.parametrize("top_k,top_p,min_p", [(5000, 1.0, 0.0), (5000, 0.9, 0.0), (40000, 0.5, 0.01), (0, 0.97, 0.0), (0, 0.97, 0.02), (0, 0.97, 0.3),
                                              (0, 1.0, 1e-4), (511, 0.99, 0.0), (513, 0.99, 0.0)])
@pytest.mark.parametrize("steps", [0, 2, 64])
def test_many_tokens_kept(top_k, top_p, min_p, steps):
    """More than a list of 4,096 holds, by each filter and by two; logits in steps of 1 / steps, so that thousands tie at the border."""
    rng = np.random.default_rng(steps + top_k)
    n, vocab = 6, 50001
    x = (rng.standard_normal((n, vocab)) * 0.8).astype(np.float32)
    if steps:
        x = np.round(x * steps) / steps
    check(x.astype(np.float32), [0.9] * n, [0.0, 0.2, 0.5, 0.8, 0.999, 1.0], [top_k] * n, [top_p] * n, [min_p] * n)


@pytest.mark.parametrize("make", ["noise", "high", "half", "spike", "pit", "slope"])
@pytest.mark.parametrize("spread", [1e-5, 0.01, 0.2, 1.0])
def test_rows_that_are_nearly_flat(spread, make):
    """Nearly everything counts for something, and top-p's border lies far down: rows far from zero, with masked halves, with one logit far above
    or below the others, with a long even slope."""
    rng = np.random.default_rng(int(spread * 1e6))
    n, vocab = 8, 40003
    x = rng.standard_normal((n, vocab)) * spread
    if make == "high":
        x += 500.0
    if make == "half":
        x[:, ::2] = -np.inf
    if make == "spike":
        x[:, 17] += 4.0
    if make == "pit":
        x[:, 17] -= 1e6
    if make == "slope":
        x = np.linspace(0.0, spread, vocab)[None].repeat(n, 0)
    top_p = [0.01, 0.3, 0.95, 0.999, 0.99999, 0.3, 0.95, 0.999]
    check(x.astype(np.float32), [1.0, 0.7, 1.0, 1.3, 1.0, 0.7, 1.0, 1.3], [0.1, 0.9, 0.5, 0.99, 1.0, 0.0, 0.7, 0.3], [0] * n, top_p,
          [0.0] * 5 + [0.5, 0.9, 0.01])


@pytest.mark.parametrize("vocab", [255, 16385, 65536])
def test_equal_logits_count_in_the_order_of_ids(vocab):
    """All logits alike (as -0 and 0 are): k of them are the first k, a share p of them the first ceil(p n)."""
    x = np.zeros((6, vocab), dtype=np.float32)
    x[:, 1::2] = -0.0
    u = [0.0, 0.999, 0.5, 0.999, 1.0, 0.25]
    k, p, m = [5, 5, 0, 0, 100, 0], [1.0, 1.0, 0.5, 0.25, 0.5, 1.0], [0, 0, 0, 0, 0, 1.0]
    check(x, [1.0, 3.0, 1.0, 0.5, 1.0, 1.0], u, k, p, m)


def test_extreme_logits_and_temperatures():
    vocab = 3000
    rng = np.random.default_rng(3)
    x = rng.standard_normal((10, vocab)).astype(np.float32)
    x[0, 17] = np.inf
    x[1] = np.nan
    x[2] = -np.inf
    x[3] *= 1e30
    x[4, 5] = 3e38
    x[4, 6] = -3e38
    x[5] = x[5] * 1e-3 + 1e6
    temperature = [1.0, 1.0, 1.0, 1e28, 1.0, 1e-3, 1e-40, 1e30, 0.0, -1.0]
    check(x, temperature, [0.3] * 10, [40] * 10, [0.9] * 10, [0.0] * 10)
    temperature[8:] = [float("inf"), 3.4e38]
    for k, p, m in ((0, 0.9, 0.0), (0, 0.9, 0.01), (0, 1.0, 0.01), (600, 1.0, 0.0)):
        check(x, temperature, [0.3] * 10, [k] * 10, [p] * 10, [m] * 10)


@pytest.mark.parametrize("vocab", [1003, 16384, 65536])
def test_a_row_without_filters_picks_as_without_them(vocab):
    """Whatever rows beside it ask for: its sums are those of the kernel without filters."""
    rng = np.random.default_rng(9)
    n = 40
    x = rng.standard_normal((n, vocab)).astype(np.float32) * 2
    u, t = rng.random(n).astype(np.float32), rng.uniform(0.5, 1.2, n).astype(np.float32)
    t[3] = 0.0
    alone = run(x, t, u)
    off = run(x, t, u, [0, vocab] * (n // 2), [1.0] * n, [0.0] * n)
    assert off == alone
    k = [0 if r % 2 else 3 for r in range(n)]
    mixed = run(x, t, u, top_k=k)
    assert mixed[1::2] == alone[1::2]
    assert all(mixed[r] in np.argsort(-x[r], kind="stable")[:3] for r in range(0, n, 2))


@pytest.mark.parametrize("offset", [1, 2, 3])
def test_rows_at_any_alignment(offset):
    vocab, n = 5003, 7
    rng = np.random.default_rng(offset)
    x = rng.standard_normal((n, vocab)).astype(np.float32) * 3
    room = torch.full((n * vocab + 8,), float("inf"), device=DEV)     # (what stands around the rows would win)
    rows = room[offset:offset + n * vocab].view(n, vocab)
    rows.copy_(torch.from_numpy(x))
    u = rng.random(n).astype(np.float32)
    out = torch.empty(n, dtype=torch.int32, device=DEV)
    ops().sample_rows(rows, torch.ones(n, device=DEV), torch.from_numpy(u).to(DEV), out, top_p=torch.full((n,), 0.9, device=DEV))
    assert out.cpu().tolist() == [plain.pick(x[r], 1.0, float(u[r]), 0, 0.9) for r in range(n)]


def test_draws_follow_the_filtered_distribution():
    n = 4000
    x = np.tile(np.array([[0.0, 1.0, 2.0, -1.0, 0.5, 1.5]], dtype=np.float32), (n, 1))
    u = np.random.default_rng(1).random(n).astype(np.float32)
    got = np.bincount(run(x, [1.0] * n, u, top_k=[4] * n), minlength=6) / n
    w = np.where(np.arange(6)[None] != 3, np.exp(x[0]), 0)[0]
    w[0] = 0
    # four standard deviations of a frequency among 4,000 draws: 4 sqrt(1/4 / 4000)
    assert np.abs(got - w / w.sum()).max() < 4 * 0.5 / np.sqrt(n)


def test_the_longest_row():
    vocab = 1 << 19
    rng = np.random.default_rng(11)
    x = np.zeros((2, vocab), dtype=np.float32)
    x[1] = rng.standard_normal(vocab)
    check(x, [1.0, 2.0], [0.75, 0.5], [0, 0], [0.5, 0.99], [0.0, 0.0])
    with pytest.raises(ops().KernelArgumentError, match="at most"):
        one = torch.zeros(1, device=DEV)
        ops().sample_rows(torch.zeros(1, vocab + 1, device=DEV), one + 1, one, torch.zeros(1, dtype=torch.int32, device=DEV), top_p=one)


def test_replays_follow_what_changes_on_the_device():
    vocab, n = 2048, 5
    g = torch.Generator(device=DEV).manual_seed(4)
    x, t = torch.randn(n, vocab, generator=g, device=DEV), torch.full((n,), 0.9, device=DEV)
    u, k = torch.rand(n, generator=g, device=DEV), torch.full((n,), 20, dtype=torch.int32, device=DEV)
    p = torch.full((n,), 0.8, device=DEV)
    out = torch.zeros(n, dtype=torch.int32, device=DEV)
    ops().sample_rows(x, t, u, out, top_k=k, top_p=p)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops().sample_rows(x, t, u, out, top_k=k, top_p=p)
    for i in range(4):
        x.normal_(generator=g)
        u.uniform_(generator=g)
        k.fill_(i * 15)
        graph.replay()
        torch.cuda.synchronize()
        want = [plain.pick(x[r].cpu().numpy(), float(np.float32(0.9)), float(u[r]), i * 15, 0.8) for r in range(n)]
        assert out.cpu().tolist() == want


def test_refusals():
    x, one = torch.zeros(2, 8, device=DEV), torch.ones(2, device=DEV)
    out, k = torch.zeros(2, dtype=torch.int32, device=DEV), torch.ones(2, dtype=torch.int32, device=DEV)
    bad = ops().KernelArgumentError
    for kw in ({"top_k": one}, {"top_k": k[:1]}, {"top_p": k}, {"min_p": one[:1]}, {"top_p": one.cpu()}):
        with pytest.raises(bad):
            ops().sample_rows(x, one, one, out, **kw)
    with pytest.raises(bad, match="not contiguous"):
        ops().sample_rows(torch.zeros(8, 2, device=DEV).t(), one, one, out, top_k=k)
    ops().sample_rows(x[:0], one[:0], one[:0], out[:0], top_k=k[:0])          # no rows: nothing to do


def test_generate_draws_among_the_likeliest(loud_model_dirs):
    """One token left is the greedy one whatever the seed, and a request's draws do not depend on who runs beside it."""
    from imparo_amd import generate
    d = loud_model_dirs["A"]
    prompts = [[5, 17, 3], [9, 9, 30, 2]]
    greedy = generate(d, prompts, max_tokens=8, dtype="float32", page_size=8)
    for only in ({"top_k": 1}, {"top_p": 1e-6}, {"min_p": 1.0}):
        assert generate(d, prompts, max_tokens=8, dtype="float32", page_size=8, temperature=1.5, seed=3, **only) == greedy
    free = generate(d, prompts, max_tokens=8, dtype="float32", page_size=8, temperature=5.0, seed=3)
    some = generate(d, prompts, max_tokens=8, dtype="float32", page_size=8, temperature=5.0, seed=3, top_k=3)
    assert some != free and some != greedy
    assert generate(d, prompts[:1], max_tokens=8, dtype="float32", page_size=8, temperature=5.0, seed=3, top_k=3) == some[:1]
    assert generate(d, prompts, max_tokens=8, dtype="float32", page_size=8, temperature=5.0, seed=3, top_k=3, overlap=False) == some


@pytest.mark.parametrize("vocab", [16385, 65536])
@pytest.mark.parametrize("level", [0.1, 1.1, 4.9, -11.762, 1e36])
def test_rows_whose_largest_logits_are_all_alike(level, vocab):
    """Every thread's largest logit is the row's, a number whose multiples round (or overflow): constant rows under top-p, alone and with
    min-p, and constant rows of which a part is masked, hardly likely or far below; each behind a row of another kind, with other bins."""
    rng = np.random.default_rng(vocab)
    rows = []
    for rest in (None, -np.inf, level - 60, level - 1e4):
        x = np.full(vocab, level)
        if rest is not None:
            x[rng.random(vocab) < 0.3] = rest
        rows += [rng.standard_normal(vocab) * 2, x]
    x = np.stack(rows).astype(np.float32)
    n = len(rows)
    for p, m in ((0.5, 0.0), (0.95, 0.3), (1e-6, 0.0), (1.0 - 2.0 ** -20, 1.0)):
        check(x, [1.0, 0.7] * (n // 2), [0.3, 0.0, 0.9, 0.3, 0.1, 0.7, 0.5, 0.999], [0] * n, [0.9, p] * (n // 2), [0.0, m] * (n // 2))


@pytest.mark.parametrize("vocab", [1003, (1 << 19) + 1])
def test_filters_of_greedy_rows_filter_nothing(vocab, monkeypatch):
    """Beside rows that are drawn without filters, whose step goes through the kernel without filters and takes rows of any length."""
    from imparo_amd.sampling.sampler import NO_FILTERS, Sampler
    from imparo_amd.kernels import ops as o
    rng = np.random.default_rng(5)
    x = rng.standard_normal((4, vocab)).astype(np.float32)
    seen, rows = [], o.sample_rows
    monkeypatch.setattr(o, "sample_rows", lambda *a, **filters: seen.append(filters) or rows(*a, **filters))
    sampler = Sampler(DEV)
    t, u = [0.0, 0.9, -1.0, 0.7], [0.5, 0.25, 0.5, 0.75]
    logits = torch.from_numpy(x).to(DEV)
    got = sampler.pick(logits, t, u, [(5, 1.0, 0.0), NO_FILTERS, (0, 0.9, 0.1), NO_FILTERS])
    assert got == sampler.pick(logits, t, u) and seen == [{}, {}]
    assert got[0] == int(x[0].argmax()) and got[2] == int(x[2].argmax())
    if vocab < 1 << 19:
        got = sampler.pick(logits, t, u, [NO_FILTERS, (1, 1.0, 0.0), NO_FILTERS, NO_FILTERS])
        assert got[1] == int(x[1].argmax()) and list(seen[2]) == ["top_k", "top_p", "min_p"]


@pytest.mark.parametrize("vocab", [1003, 16385, 65536])
@pytest.mark.parametrize("level", [float(np.finfo(np.float32).min), -3.2e38, float(np.finfo(np.float32).max)])
def test_rows_at_the_ends_of_float32(level, vocab):
    """A row all of whose logits are a mask's lowest value (or the largest one) picks among them as any row of equal logits does, also
    where a few are masked by minus infinity; a row with some such masks among ordinary logits leaves them out."""
    rng = np.random.default_rng(vocab)
    x = np.full((6, vocab), level, dtype=np.float32)
    x[1, rng.random(vocab) < 0.3] = -np.inf
    x[2:4] = np.where(rng.random((2, vocab)) < 0.5, min(level, -level), rng.standard_normal((2, vocab)) * 2).astype(np.float32)
    x[4, 7] = np.nan
    u, t = [0.0, 0.6, 0.3, 0.9, 0.999, 1.0], [1.0, 0.7, 1.0, 0.5, 1e3, 1.0]
    for k, p, m in ((0, 0.9, 0.0), (0, 0.5, 0.3), (0, 1.0, 0.5), (400, 1.0, 0.0), (700, 0.9, 0.0), (400, 0.5, 1.0)):
        check(x, t, u, [k] * 6, [p] * 6, [m] * 6)
