"""Decode attention of rows that share a prefix against the plain form in 64 bits."""
import math

import numpy as np
import pytest
import torch

import plain_continuations as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def ops():
    from imparo_amd.kernels import ops as o
    return o


def ints(a):
    return torch.tensor(np.asarray(a, dtype=np.int32), device=DEV)


class Batch:
    """Groups of (shared keys, [keys behind them, row by row]); rows in no group as (None, [keys]). Pages in no order, everything
    that no row sees poisoned with NaN, one row of tokens that is not listed, the list in no order of tokens."""

    def __init__(self, groups, heads, kv, dim, page, seed=0, spread=1.5):
        rng = np.random.default_rng(seed)
        g = torch.Generator().manual_seed(seed)
        self.page, self.heads = page, heads
        total = sum(-(-(s or 0) // page) + sum(-(-((s or 0) + b) // page) + 1 for b in own) for s, own in groups) + 3
        free = iter(rng.permutation(total).tolist())
        nan = float("nan")
        self.k = torch.full((total, kv, page, dim), nan, dtype=torch.bfloat16)
        self.v = torch.full((total, kv, dim, page), nan, dtype=torch.bfloat16)

        def fill(p, upto):
            self.k[p, :, :upto] = torch.randn(kv, upto, dim, generator=g).to(torch.bfloat16)
            self.v[p, :, :, :upto] = torch.randn(kv, dim, upto, generator=g).to(torch.bfloat16)

        tables, positions, self.group_start, self.shared = [], [], [0], []
        for shared, own in groups:
            s = shared or 0
            whole = [next(free) for _ in range(s // page)]
            for p in whole:
                fill(p, page)
            part = next(free) if s % page else None          # the page the shared keys end in: its own copy for every row
            if part is not None:
                fill(part, s % page)
            for j, b in enumerate(own):
                table = list(whole)
                if b < 0:                                      # a row inside the prefix
                    if part is not None:
                        table.append(part)
                elif part is not None:
                    mine = part if j == 0 else next(free)
                    if mine != part:
                        self.k[mine], self.v[mine] = self.k[part], self.v[part]
                    table.append(mine)
                if b > 0:
                    while len(table) * page < s + b:
                        table.append(next(free))
                    for key in range(s, s + b):
                        p = table[key // page]
                        self.k[p, :, key % page] = torch.randn(kv, dim, generator=g).to(torch.bfloat16)
                        self.v[p, :, :, key % page] = torch.randn(kv, dim, generator=g).to(torch.bfloat16)
                tables.append(table)
                positions.append(s + b - 1)
            if shared is not None:
                self.group_start.append(len(tables))
                self.shared.append(s)
        self.n = n = len(tables)
        width = max(len(t) for t in tables) + 1
        self.order = rng.permutation(n)                       # listed row i is row order[i], its token also order[i]
        self.tables = [None] * n
        self.positions = [0] * n
        for i, r in enumerate(self.order):
            self.tables[r], self.positions[r] = tables[i], positions[i]
        self.q = (torch.randn(n + 1, heads, dim, generator=g) * spread).to(torch.bfloat16)
        self.table = np.full((n + 1, width), -1, dtype=np.int32)
        for r in range(n):
            self.table[r, :len(self.tables[r])] = self.tables[r]
        self.max_shared = max(self.shared, default=0)
        in_group = {i: s for g, s in enumerate(self.shared) for i in range(self.group_start[g], self.group_start[g + 1])}
        self.max_own = max(max(positions[i] + 1 - in_group.get(i, 0), 0) for i in range(n))
        self.max_group = max((b - a for a, b in zip(self.group_start, self.group_start[1:])), default=0)
        self.scale = dim ** -0.5

    def run(self, window=None, stretch=0, scale=None):
        n, heads, dim = self.q.shape
        kv = self.k.shape[1]
        bounds = dict(max_shared=self.max_shared + stretch, max_own=self.max_own + stretch, max_group=self.max_group + stretch)
        parts = ops().attention_shared_parts(self.n, heads, kv, dim, len(self.shared), bounds["max_group"], bounds["max_shared"],
                                             bounds["max_own"])
        nan = float("nan")
        out = torch.full((n, heads * dim), 7.0, dtype=torch.bfloat16, device=DEV)
        part_o = torch.full((self.n, heads, parts, dim), nan, device=DEV)
        part_ml = torch.full((self.n, heads, parts, 2), nan, device=DEV)
        back = ops().attention_decode_shared(
            self.q.to(DEV), self.k.to(DEV), self.v.to(DEV), out, part_o, part_ml, ints(self.order), self.n, ints(self.group_start),
            ints(self.shared), ints(np.arange(n)), ints(self.positions + [0]), ints(self.table), scale or self.scale, window, **bounds)
        assert back is out
        assert torch.equal(out[self.n].cpu(), torch.full((heads * dim,), 7.0, dtype=torch.bfloat16))
        return out[:self.n].cpu()

    def check(self, window=None, stretch=0, scale=None):
        got = self.run(window, stretch, scale).double()
        want, bound = plain.attend(self.q[:self.n], self.k, self.v, self.tables, self.positions, scale or self.scale, window)
        over = (got - want).abs() - bound
        assert not got.isnan().any() and bool((over <= 0).all()), (float(over.max()), float((got - want).abs().max()))


@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("heads,kv", [(4, 4), (6, 2), (8, 1)])
def test_heads_of_all_sizes(dim, heads, kv):
    Batch([(200, [3, 40, 1, 70])], heads, kv, dim, 32, seed=dim).check()


@pytest.mark.parametrize("page", [16, 32, 64, 256])
@pytest.mark.parametrize("shared", [1, 15, 16, 31, 33, 64, 127, 128, 129, 300, 512, 700])
def test_where_the_shared_keys_end(page, shared):
    Batch([(shared, [1, 2, 31, 33, 64])], 4, 2, 32, page, seed=shared).check()


@pytest.mark.parametrize("groups", [
    [(100, [1])],                                              # one row alone in its group
    [(0, [5, 1, 300])],                                        # a group that shares nothing
    [(None, [1, 17, 290])],                                    # rows in no group
    [(64, [0, 0])],                                            # no keys of their own
    [(64, [4, 9]), (None, [7]), ],                             # the last rows are in no group
    [(40, [3] * 9), (333, [1, 2, 70]), (16, [500])],
    [(257, [1] * 70)],                                         # more queries than a block's tile
    [(90, [-40, -89, 5, -90])],                                # rows inside the prefix, one that sees nothing
])
@pytest.mark.parametrize("stretch", [0, 1000])
def test_groups(groups, stretch):
    Batch(groups, 4, 2, 64, 16, seed=5).check(stretch=stretch)


@pytest.mark.parametrize("heads,kv", [(32, 1), (33, 1), (48, 1), (70, 2)])
def test_many_heads_a_kv_head(heads, kv):
    Batch([(75, [1, 30, 9])], heads, kv, 32, 16, seed=heads).check()


@pytest.mark.parametrize("window", [1, 7, 32, 100, 260, 10000])
def test_windows(window):
    Batch([(290, [1, 40, 128, 300]), (20, [3, 3])], 4, 2, 64, 32, seed=window).check(window=window)


@pytest.mark.parametrize("heads,kv,dim,page", [(4, 2, 64, 32), (4, 2, 48, 64), (48, 1, 64, 64), (48, 1, 128, 16), (70, 2, 80, 128)])
@pytest.mark.parametrize("groups,window", [([(210, [-150, -60, 4, 30])], None), ([(290, [1, 40, 128])], 100), ([(290, [-200, -120, 3, 200])], 150)])
@pytest.mark.parametrize("scale", [None, -0.2])
def test_values_that_are_not_finite_reach_only_rows_that_see_them(groups, window, scale, heads, kv, dim, page):
    """Among the shared keys, where some rows of a group see what others do not: an infinity, then one of the other sign and a NaN."""
    b = Batch(groups, heads, kv, dim, page, seed=dim)
    table = b.tables[int(np.argmax(b.positions))]
    for key, d, value in ((100, 1, float("inf")), (110, 4, float("-inf")), (190, 2, float("nan")), (200, 3, float("-inf")), (206, 3, float("inf"))):
        if key < groups[0][0] // page * page:
            b.v[table[key // page], :, d, key % page] = value
    got = b.run(window, scale=scale).double()
    want, bound = plain.attend(b.q[:b.n], b.k, b.v, b.tables, b.positions, scale or b.scale, window)
    fine = want.isfinite()
    assert not fine.all() and fine.view(b.n, heads, dim).all(dim=2).any()          # rows of either kind
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[want.isinf()], want[want.isinf()])
    over = (got - want).abs()[fine] - bound[fine]
    assert bool((over <= 0).all()), float(over.max())


@pytest.mark.parametrize("spread,scale", [(0.0, None), (30.0, None), (1.5, -0.2), (1.5, 1e-3)])
def test_flat_and_steep_scores(spread, scale):
    """Queries of zero (all keys alike), scores far apart (the reference of the exponentials moves from tile to tile), and scales of either sign."""
    Batch([(400, [60, 3, 129])], 4, 2, 64, 32, seed=2, spread=spread).check(scale=scale)


@pytest.mark.parametrize("seed", range(12))
def test_batches_of_any_make(seed):
    rng = np.random.default_rng(1000 + seed)
    kv = int(rng.choice([1, 2, 3]))
    groups = [(None if rng.random() < 0.2 else int(rng.integers(0, 400)), [int(b) for b in rng.integers(1, 200, rng.integers(1, 9))])
              for _ in range(rng.integers(1, 6))]
    groups = [g for g in groups if g[0] is not None] + [g for g in groups if g[0] is None]
    b = Batch(groups, kv * int(rng.integers(1, 20)), kv, int(rng.choice([16, 32, 48, 64, 80, 96, 112, 128])),
              int(rng.choice([16, 32, 64, 128])), seed=seed)
    b.check(window=None if rng.random() < 0.6 else int(rng.integers(1, 300)), stretch=int(rng.choice([0, 100])))


def test_a_long_prefix():
    Batch([(4500, [100, 600, 1])], 4, 2, 64, 64, seed=8).check()


def test_agrees_with_attention_of_each_row_by_itself():
    """The same inputs through the kernel that reads everything a row: both inside the bound of the plain form."""
    b = Batch([(512, [30, 64, 5, 200])], 8, 2, 64, 64, seed=3)
    n, heads, dim = b.q.shape
    split = ops().decode_split()
    context = max(b.positions) + 1
    n_splits = -(-context // split)
    out = torch.zeros(n, heads * dim, dtype=torch.bfloat16, device=DEV)
    ops().attention_decode(b.q.to(DEV), b.k.to(DEV), b.v.to(DEV), out, torch.empty(b.n * heads * n_splits * dim, device=DEV),
                           torch.empty(b.n * heads * n_splits * 2, device=DEV), ints(b.order), b.n, ints(np.arange(n)),
                           ints(b.positions + [0]), ints(b.table), b.scale, None, context)
    _, bound = plain.attend(b.q[:b.n], b.k, b.v, b.tables, b.positions, b.scale)
    assert bool(((out[:b.n].cpu().double() - b.run().double()).abs() <= 2 * bound).all())


def test_replays_follow_what_changes_on_the_device():
    b = Batch([(200, [40, 50, 60, 70])], 8, 2, 64, 32, seed=6)
    n, heads, dim = b.q.shape
    bounds = dict(max_shared=200, max_own=300, max_group=4)      # (the last replay shares nothing)
    parts = ops().attention_shared_parts(b.n, heads, 2, dim, 1, 4, 200, 300)
    out = torch.zeros(n, heads * dim, dtype=torch.bfloat16, device=DEV)
    part_o, part_ml = torch.empty(b.n, heads, parts, dim, device=DEV), torch.empty(b.n, heads, parts, 2, device=DEV)
    q, k, v, shared, positions = b.q.to(DEV), b.k.to(DEV), b.v.to(DEV), ints([200]), ints(b.positions + [0])
    args = (q, k, v, out, part_o, part_ml, ints(b.order), b.n, ints([0, 4]), shared, ints(np.arange(n)), positions, ints(b.table),
            b.scale, None)
    ops().attention_decode_shared(*args, **bounds)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops().attention_decode_shared(*args, **bounds)
    for i, (s, back) in enumerate([(200, 0), (192, 3), (96, 30), (0, 0)]):
        shared.fill_(s)
        now = [p - back for p in b.positions]
        positions.copy_(ints(now + [0]))
        part_o.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        want, bound = plain.attend(b.q[:b.n], b.k, b.v, b.tables, now, b.scale)
        assert bool(((out[:b.n].cpu().double() - want).abs() <= bound).all()), i


def test_a_cache_of_more_than_2_to_32_elements():
    """Pages at both ends of a cache whose last elements lie past 32 bits."""
    b = Batch([(130, [40, 3, 90])], 8, 8, 128, 64, seed=12)
    low = b.run()
    n_pages = (1 << 32) // (8 * 64 * 128) + b.k.shape[0]
    shift = n_pages - b.k.shape[0]
    k = torch.empty(n_pages, 8, 64, 128, dtype=torch.bfloat16, device=DEV)
    v = torch.empty(n_pages, 8, 128, 64, dtype=torch.bfloat16, device=DEV)
    k[shift:], v[shift:] = b.k.to(DEV), b.v.to(DEV)
    n, heads, dim = b.q.shape
    bounds = dict(max_shared=b.max_shared, max_own=b.max_own, max_group=b.max_group)
    parts = ops().attention_shared_parts(b.n, heads, 8, dim, 1, b.max_group, b.max_shared, b.max_own)
    out = torch.zeros(n, heads * dim, dtype=torch.bfloat16, device=DEV)
    table = np.where(b.table >= 0, b.table + shift, -1)
    ops().attention_decode_shared(b.q.to(DEV), k, v, out, torch.empty(b.n, heads, parts, dim, device=DEV),
                                  torch.empty(b.n, heads, parts, 2, device=DEV), ints(b.order), b.n, ints(b.group_start), ints(b.shared),
                                  ints(np.arange(n)), ints(b.positions + [0]), ints(table), b.scale, None, **bounds)
    assert torch.equal(out[:b.n].cpu(), low)                  # (the same work whatever the pages' numbers: the same bits)


def test_two_streams_with_scratch_of_their_own():
    a, b = Batch([(300, [30, 64, 5])], 8, 2, 64, 32, seed=3), Batch([(200, [3, 164, 50])], 8, 2, 64, 32, seed=4)
    want = a.run(), b.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got_b = b.run()
    got_a = a.run()
    torch.cuda.synchronize()
    assert torch.equal(got_a, want[0]) and torch.equal(got_b, want[1])


def test_refusals():
    b = Batch([(32, [4, 4])], 4, 2, 64, 32, seed=1)
    n, heads, dim = b.q.shape
    bad = ops().KernelArgumentError
    good = dict(q=b.q.to(DEV), k_cache=b.k.to(DEV), v_cache=b.v.to(DEV),
                out=torch.zeros(n, heads * dim, dtype=torch.bfloat16, device=DEV), part_o=torch.zeros(4096 * 8, device=DEV),
                part_ml=torch.zeros(4096, device=DEV), rows=ints(b.order), n_rows=2, group_start=ints([0, 2]), shared=ints([32]),
                seg_start=ints(np.arange(n)), positions=ints(b.positions + [0]), block_table=ints(b.table), scale=0.1, window=None,
                max_shared=32, max_own=8, max_group=2)
    ops().attention_decode_shared(**good)
    for name, value in [("q", good["q"].float()), ("k_cache", good["k_cache"].float()), ("out", good["out"][:1]),
                        ("v_cache", good["v_cache"].transpose(2, 3)), ("n_rows", 3), ("n_rows", -1), ("window", 0), ("window", -4),
                        ("group_start", ints([])), ("shared", ints([1, 2])), ("block_table", ints(b.table)[:1]),
                        ("positions", ints([0])), ("part_o", torch.zeros(16, device=DEV)), ("part_ml", torch.zeros(4, device=DEV)),
                        ("max_own", -1), ("max_shared", (1 << 30) + 1), ("rows", ints(b.order).long()), ("q", good["q"].cpu()),
                        ("part_o", torch.zeros(4096 * 8 + 4, device=DEV)[1:])]:
        with pytest.raises(bad):
            ops().attention_decode_shared(**{**good, name: value})
    out = torch.full_like(good["out"], 3.0)
    ops().attention_decode_shared(**{**good, "out": out, "n_rows": 0})
    assert bool((out == 3.0).all())


@pytest.mark.parametrize("heads,kv,dim,page", [(4, 2, 64, 32), (4, 2, 48, 64), (48, 1, 128, 16), (70, 2, 80, 128)])
@pytest.mark.parametrize("where", ["query", "key alone", "key among others", "key far down", "infinite key", "value far down"])
@pytest.mark.parametrize("scale", [None, -0.2])
def test_what_is_not_a_number_in_what_a_row_sees(where, scale, heads, kv, dim, page):
    """In a query, in keys (the only one of a part, one of many, one whose part weighs nothing beside another) and in a value whose part
    weighs nothing: no finite result where the plain form has none, and no other row touched."""
    b = Batch([(290, [1, 40, 1]), (40, [3, 2]), (None, [70])], heads, kv, dim, page, seed=dim)
    r, nan = int(b.order[0]), float("nan")
    place = lambda key: (b.tables[r][key // page], key % page)
    if where == "query":
        b.q[r, 1, 5] = nan
    if where == "key alone":
        p, s = place(290)
        b.k[p, :, s] = nan
    if where == "key among others":
        p, s = place(100)
        b.k[p, 0, s, 7] = nan
    if where == "infinite key":                                # (an infinite score, or one of minus infinity, as the query's sign has it)
        p, s = place(100)
        b.k[p, :, s, 3] = float("inf")
    if where.endswith("far down"):                             # all of the row's weight in the first head on its last key
        p, s = place(290)
        b.k[p, 0, s] = 30.0 * torch.sign(b.q[r, 0]) * (-1 if scale else 1)
        p, s = place(5)
        if where == "key far down":
            b.k[p, 0, s, 7] = nan
        else:
            b.v[p, 0, 2, s] = nan
    got = b.run(scale=scale).double()
    want, bound = plain.attend(b.q[:b.n], b.k, b.v, b.tables, b.positions, scale or b.scale)
    assert want.isnan().any() and not want.isnan().all()
    assert torch.equal(got.isnan(), want.isnan()), (int(got.isnan().sum()), int(want.isnan().sum()))
    over = torch.where(want.isnan(), 0.0, (got - want).abs() - torch.where(bound.isnan(), math.inf, bound))
    assert bool((over <= 0).all()), float(over.max())


@pytest.mark.parametrize("heads,kv", [(4, 2), (48, 1)])
@pytest.mark.parametrize("broken", [{"max_own": 1}, {"max_own": 0}, {"max_shared": 64}, {"max_shared": 0}, {"max_group": 1}, {"max_group": 0}])
def test_rows_past_a_bound_are_not_numbers(broken, heads, kv):
    """Bounds are about numbers on the device, which the host cannot look at. Over scratch that holds what an earlier call might have left there, a
    row past a bound is NaN as a whole, or right where the launch reached all its keys; the others are right."""
    dim, page = 64, 32
    b = Batch([(300, [200, 1, 3] + [2] * 60), (40, [3, 180]), (None, [1, 90])], heads, kv, dim, page, seed=heads)
    bounds = {**dict(max_shared=b.max_shared, max_own=b.max_own, max_group=b.max_group), **broken}
    n = b.n + 1
    parts = ops().attention_shared_parts(b.n, heads, kv, dim, len(b.shared), bounds["max_group"], bounds["max_shared"], bounds["max_own"])
    out = torch.full((n, heads * dim), 7.0, dtype=torch.bfloat16, device=DEV)
    part_o, part_ml = torch.full((b.n, heads, parts, dim), 3.0, device=DEV), torch.full((b.n, heads, parts, 2), 5.0, device=DEV)
    ops().attention_decode_shared(b.q.to(DEV), b.k.to(DEV), b.v.to(DEV), out, part_o, part_ml, ints(b.order), b.n, ints(b.group_start),
                                  ints(b.shared), ints(np.arange(n)), ints(b.positions + [0]), ints(b.table), b.scale, None, **bounds)
    got = out[:b.n].cpu().double()
    want, bound = plain.attend(b.q[:b.n], b.k, b.v, b.tables, b.positions, b.scale)
    right, lost = ((got - want).abs() <= bound).all(dim=1), got.isnan().all(dim=1)
    assert bool((right | lost).all()), (~(right | lost)).nonzero().flatten().tolist()
    in_group = [(g, i - a) for g, (a, e) in enumerate(zip(b.group_start, b.group_start[1:])) for i in range(a, e)]
    for i in range(b.n):                                       # listed row i
        g, place = in_group[i] if i < len(in_group) else (None, 0)
        shared = b.shared[g] if g is not None else 0
        own = b.positions[b.order[i]] + 1 - shared
        if shared <= bounds["max_shared"] and own <= bounds["max_own"] and (not shared or place < bounds["max_group"]):
            assert bool(right[b.order[i]]), i
    assert bool(lost.any())


def with_values_of_one(b):
    b.v = torch.where(b.v.isnan(), b.v, torch.ones_like(b.v))
    return b


@pytest.mark.parametrize("heads,kv,dim,page", [(4, 2, 64, 32), (4, 2, 48, 64), (48, 1, 64, 64), (48, 1, 128, 16), (70, 2, 80, 128)])
@pytest.mark.parametrize("spread", [0.5, 5.0, 30.0])
def test_values_that_are_all_alike_come_out_as_they_are(spread, heads, kv, dim, page):
    """A sum of weights over the sum of the same weights, whatever a weight was rounded to: 1 off by no more than float32 sums of some hundred
    terms are (500 times 1.5e-7, and 500 2^-24), and bfloat16's nearest number to that is 1 (the next one below lies 2^-8 away)."""
    b = with_values_of_one(Batch([(300, [1, 40, 170]), (0, [33, 260])], heads, kv, dim, page, seed=dim, spread=spread))
    assert torch.equal(b.run(), torch.ones(b.n, heads * dim, dtype=torch.bfloat16))


@pytest.mark.parametrize("heads,kv,dim,page", [(8, 2, 64, 64), (48, 1, 64, 16), (48, 1, 128, 128)])
@pytest.mark.parametrize("groups,low,high", [([(128, [1] * 8)], 3, 70), ([(None, [64] * 8)], 3, 40)])
def test_the_same_where_one_key_of_a_later_tile_has_nearly_all_the_weight(groups, low, high, heads, kv, dim, page):
    """Its weight is then any number up to 2^8 (the reference of the exponentials stays with the first tile's largest score, at `low`), not 1."""
    b = with_values_of_one(Batch(groups, heads, kv, dim, page, seed=dim))
    octaves = torch.linspace(4.0, 7.9, (b.n + 1) * heads).view(b.n + 1, heads, 1)          # of the score at `high` above that at `low`
    b.q = (octaves / (dim * b.scale * math.log2(math.e)) * torch.ones(dim)).to(torch.bfloat16)
    b.k = torch.where(b.k.isnan(), b.k, -torch.ones_like(b.k))
    for table in b.tables:
        b.k[table[low // page], :, low % page] = 0.0
        b.k[table[high // page], :, high % page] = 1.0
    assert torch.equal(b.run(), torch.ones(b.n, heads * dim, dtype=torch.bfloat16))


@pytest.mark.parametrize("heads,kv", [(8, 2), (48, 1)])
def test_a_nan_that_all_rows_see_costs_nothing(heads, kv):
    """One value of a shared prefix: the products pass it on by themselves. (Sums made anew, key by key, took a hundred times the call's time.)"""
    b = Batch([(4096, [1, 2, 3, 4])], heads, kv, 64, 64, seed=1)
    n, dim = b.n + 1, 64
    bounds = dict(max_shared=b.max_shared, max_own=b.max_own, max_group=b.max_group)
    parts = ops().attention_shared_parts(b.n, heads, kv, dim, 1, *(bounds[k] for k in ("max_group", "max_shared", "max_own")))
    out = torch.zeros(n, heads * dim, dtype=torch.bfloat16, device=DEV)
    part_o, part_ml = torch.empty(b.n, heads, parts, dim, device=DEV), torch.empty(b.n, heads, parts, 2, device=DEV)
    k, v = b.k.to(DEV), b.v.to(DEV)
    args = (ints(b.order), b.n, ints(b.group_start), ints(b.shared), ints(np.arange(n)), ints(b.positions + [0]), ints(b.table), b.scale, None)
    q = b.q.to(DEV)

    def fastest():
        times = []
        for _ in range(8):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record()
            for _ in range(10):
                ops().attention_decode_shared(q, k, v, out, part_o, part_ml, *args, **bounds)
            end.record()
            torch.cuda.synchronize()
            times.append(begin.elapsed_time(end))
        return min(times)

    clean = fastest()
    v[b.tables[0][0], :, 3, 5] = float("nan")
    poisoned = fastest()
    rows = out[:b.n].view(b.n, heads, dim)
    assert bool(rows[:, :, 3].isnan().all()) and not rows[:, :, 4:].isnan().any()
    assert poisoned < 3 * clean, (poisoned, clean)


@pytest.mark.parametrize("heads,kv,dim,page", [(8, 2, 64, 32), (48, 1, 64, 64), (48, 1, 128, 16)])
@pytest.mark.parametrize("spread", [1.5, 5.0, 30.0])
def test_values_alike_beside_one_that_is_infinite(spread, heads, kv, dim, page):
    """At a key that two of the rows see: the others' sums are made anew, numerator and denominator out of the same weights."""
    b = with_values_of_one(Batch([(210, [-150, -60, 4, 30])], heads, kv, dim, page, seed=dim, spread=spread))
    table = b.tables[int(np.argmax(b.positions))]
    b.v[table[190 // page], :, 2, 190 % page] = float("inf")
    want = torch.ones(b.n, heads, dim, dtype=torch.bfloat16)
    want[torch.tensor(b.positions) >= 190, :, 2] = float("inf")
    got = b.run().view(b.n, heads, dim)
    # (a weight below float32's smallest number makes NaN of the infinity)
    assert torch.equal(torch.where(got[:, :, 2].isnan() & want[:, :, 2].isinf(), want[:, :, 2], got[:, :, 2]), want[:, :, 2])
    got[:, :, 2] = want[:, :, 2]
    assert torch.equal(got, want)


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 3.4e38])
def test_scales_that_are_no_numbers_are_refused(scale):
    """(The smallest scale stands for 0, and would for a NaN.)"""
    with pytest.raises(ops().KernelArgumentError):
        Batch([(32, [4, 4])], 4, 2, 64, 32, seed=1).run(scale=scale)
