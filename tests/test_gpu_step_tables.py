"""A step's tables made on the GPU against the plain form, and a run of a step's operators over them."""
import numpy as np
import pytest
import torch

import plain_continuations as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def ops():
    from imparo_amd.kernels import ops as o
    return o


def ints(a, dtype=torch.int32):
    return torch.tensor(np.asarray(a), dtype=dtype, device=DEV)


def run(lengths, new, pages, page, width, n_tokens, leader=None, shared=None, slots=True):
    n = len(lengths)
    full = lambda *s, dtype=torch.int32: torch.full(s, -7, dtype=dtype, device=DEV)
    got = {"table": full(n, width), "seg_start": full(n), "positions": full(n_tokens), "row_of_token": full(n_tokens),
           "slots": full(n_tokens, dtype=torch.int64) if slots else None, "lists": full(n), "counts": full(4)}
    ops().step_tables(ints(lengths), ints(new), ints(pages), page, got["table"], got["seg_start"], got["positions"],
                      got["row_of_token"], got["slots"], got["lists"], got["counts"], leader=None if leader is None else ints(leader),
                      shared=None if shared is None else ints(shared))
    want = plain.tables(lengths, new, pages, page, width, n_tokens, leader, shared)
    for name, t in got.items():
        if t is not None:
            assert t.cpu().tolist() == want[name], name


@pytest.mark.parametrize("page", [1, 16, 64])
@pytest.mark.parametrize("n", [1, 3, 64, 65, 300])
def test_rows_of_all_kinds(page, n):
    rng = np.random.default_rng(n + page)
    lengths = rng.integers(0, 300, n).tolist()
    new = rng.choice([0, 1, 1, 1, 2, 40, 129], n).tolist()
    need = [-(-(a + b) // page) for a, b in zip(lengths, new)]
    pages = rng.permutation(2 * sum(need) + 5)[:sum(need) + 3].tolist()
    run(lengths, new, pages, page, max(max(need), 1), sum(new) + 2)
    shared = [0] + [int(rng.integers(0, 6)) for _ in range(n - 1)]
    run(lengths, new, pages, page, max(max(need), 1) + 2, sum(new) + 2, [0] * n, shared)
    run(lengths, new, pages, page, max(max(need), 1), sum(new), list(range(n - 1, -1, -1)), shared, slots=False)


def test_leaders_of_leaders():
    """Row 2 takes three pages from row 1, which took two of them from row 0; row 3 leans on itself, 4 and 5 on one another, 6 on no row."""
    run([50, 70, 90, 20, 20, 20, 20, 10], [1, 3, 1, 1, 1, 1, 1, 1], list(range(100, 140)), 16, 8, 12, [0, 0, 1, 3, 5, 4, 99, 2],
        [0, 2, 3, 1, 1, 1, 1, 7])


@pytest.mark.parametrize("n_pages,width,n_tokens", [(0, 4, 5), (3, 4, 5), (9, 2, 5), (9, 4, 2), (9, 4, 0)])
def test_too_little_room_is_told_by_the_counts(n_pages, width, n_tokens):
    run([30, 10, 0], [1, 3, 2], list(range(20, 20 + n_pages)), 16, width, n_tokens)


def test_lengths_that_are_negative_or_long():
    run([-5, 1 << 30, 7], [-1, 1, 1], list(range(10)), 1 << 26, 20, 3)
    run([0], [5000], list(range(400)), 16, 313, 5000)


def test_most_rows():
    n = ops().STEP_TABLES_MAX_ROWS
    assert n == ops().library().imparo_step_tables_max_rows()
    run([i % 40 for i in range(n)], [1] * n, list(range(3 * n)), 16, 3, n)
    with pytest.raises(ops().KernelArgumentError, match="at most"):
        run([1] * (n + 1), [1] * (n + 1), [], 16, 1, 1)


def test_refusals_and_no_rows():
    one, table, slots = ints([1]), ints([[0]]), ints([0], torch.int64)
    good = [one, one, one, 16, table, one.clone(), one.clone(), one.clone(), slots, one.clone(), ints([0] * 4)]
    ops().step_tables(*good)
    bad = ops().KernelArgumentError
    for i, value in [(0, one.long()), (1, ints([1, 2])), (3, 12), (3, 0), (4, one), (4, ints([[0], [0]])), (5, ints([])),
                     (7, ints([1, 2])), (8, one), (9, ints([1, 2])), (10, one), (2, one.cpu())]:
        with pytest.raises(bad):
            ops().step_tables(*good[:i], value, *good[i + 1:])
    with pytest.raises(bad, match="together"):
        ops().step_tables(*good, leader=one)
    counts = ints([5] * 4)
    none = ints([])
    ops().step_tables(none, none, none, 16, ints(np.zeros((0, 1))), none, none, none, None, none, counts)
    assert counts.cpu().tolist() == [0] * 4


def test_a_step_of_continuations_on_the_device():
    """Tables, keys into the cache, attention over the shared prefix, the head's product and the picks, as a step runs them, three
    steps behind one another with lengths that move on the device; every operator's result against its plain form."""
    o = ops()
    n, heads, kv, dim, page, width, vocab = 6, 4, 2, 64, 16, 8, 500
    g = torch.Generator().manual_seed(0)
    shared_pages, leader = ints([0] + [3] * (n - 1)), ints([0] * n)
    prompt = 3 * page
    k = torch.zeros(64, kv, page, dim, dtype=torch.bfloat16, device=DEV)
    v = torch.zeros(64, kv, dim, page, dtype=torch.bfloat16, device=DEV)
    pages = ints(np.random.default_rng(0).permutation(64))
    lengths, new = ints([prompt] * n), ints([1] * n)
    head = torch.randn(vocab, heads * dim, generator=g).to(torch.bfloat16).to(DEV)
    table, start, pos = ints(np.zeros((n, width))), ints([0] * n), ints([0] * n)
    row, slots, lists, counts = ints([0] * n), ints([0] * n, torch.int64), ints([0] * n), ints([0] * 4)
    out = torch.zeros(n, heads * dim, dtype=torch.bfloat16, device=DEV)
    parts = o.attention_shared_parts(n, heads, kv, dim, 1, n, prompt, page * width - prompt)
    part_o, part_ml = torch.empty(n, heads, parts, dim, device=DEV), torch.empty(n, heads, parts, 2, device=DEV)
    q_out = torch.zeros(n, heads, dim, dtype=torch.bfloat16, device=DEV)
    logits, picks = torch.zeros(n, vocab, device=DEV), ints([0] * n)
    temperature, top_p = torch.full((n,), 0.7, device=DEV), torch.full((n,), 0.9, device=DEV)
    # the prompt's keys and values, in row 0's first pages
    k[pages[:3].long()] = torch.randn(3, kv, page, dim, generator=g).to(torch.bfloat16).to(DEV)
    v[pages[:3].long()] = torch.randn(3, kv, dim, page, generator=g).to(torch.bfloat16).to(DEV)
    for step in range(3):
        # (every row's own pages are reserved for all steps, so a row keeps its pages as it grows)
        reach = ints([prompt + page] * n) - 1
        o.step_tables(reach, new, pages, page, table, start, pos, row, slots, lists, counts, leader=leader, shared=shared_pages)
        want = plain.tables(reach.tolist(), [1] * n, pages.tolist(), page, width, n, [0] * n, shared_pages.tolist())
        assert table.cpu().tolist() == want["table"] and counts.cpu().tolist() == want["counts"] and lists.cpu().tolist() == list(range(n))
        pos.copy_(lengths)
        qkv = torch.randn(n, (heads + 2 * kv) * dim, generator=g).to(DEV)
        o.qk_norm_rope_store(qkv, None, None, 1e-5, None, pos, row, table, page, q_out, k, v, heads, kv, dim, v_transposed=True)
        o.attention_decode_shared(q_out, k, v, out, part_o, part_ml, lists, n, ints([0, n]), ints([prompt]), start, pos, table,
                                  dim ** -0.5, None, max_shared=prompt, max_own=page * width - prompt, max_group=n)
        attended, bound = plain.attend(q_out.cpu(), k.cpu(), v.cpu(), table.tolist(), pos.tolist(), dim ** -0.5)
        assert bool(((out.cpu().double() - attended).abs() <= bound).all())
        o.gemm(out, head, logits)
        u = torch.rand(n, generator=g)
        o.sample_rows(logits, temperature, u.to(DEV), picks, top_p=top_p)
        rows = logits.cpu().numpy()
        assert picks.cpu().tolist() == [plain.pick(rows[r], float(temperature[r]), float(u[r]), 0, 0.9) for r in range(n)]
        lengths += 1


def test_positions_past_32_bits():
    """Pages of one token, whose numbers are then positions: a row that grows past 2^31 names the pages there are, and no other row's."""
    full = lambda *s, dtype=torch.int32: torch.full(s, -7, dtype=dtype, device=DEV)
    top = 2 ** 31 - 1
    table, start, positions, row, slots, lists, counts = full(2, 3), full(2), full(4), full(4), full(4, dtype=torch.int64), full(2), full(4)
    ops().step_tables(ints([top, 4]), ints([3, 1]), ints([8, 6, 4, 2, 0]), 1, table, start, positions, row, slots, lists, counts)
    assert table.tolist() == [[8, 6, 4], [-1, -1, -1]] and start.tolist() == [0, 3]
    assert positions.tolist() == [top, top, top, 4] and row.tolist() == [0, 0, 0, 1] and slots.tolist() == [-1] * 4
    assert lists.tolist() == [1, 0] and counts.tolist() == [4, top, 1, 1]
