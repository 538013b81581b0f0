"""GPU tests of the page operators (``PagePool``) against their definition row by row.
Everything is compared for equality: tables, lengths, counts, free bits, status and
every slot of every cache."""
import random

import pytest
import torch

from page_model import BAD_BLOCK, BAD_ROW, BAD_SEQLEN, NO_PAGES, PageModel, assert_same

pytestmark = pytest.mark.gpu


def _setup(rows, width, nb, bs=16, hkv=2, d=64, layers=2, dtype=torch.float16, strided=False, seed=0):
    import paged_attention as pa
    g = torch.Generator().manual_seed(seed)
    k, v = [], []
    for _ in range(layers):
        if strided:       # K and V side by side in one buffer, heads before slots
            kv = torch.randn(nb, 2, hkv, bs, d, generator=g).to(dtype).cuda()
            k.append(kv[:, 0].transpose(1, 2))
            v.append(kv[:, 1].transpose(1, 2))
        else:
            k.append(torch.randn(nb, bs, hkv, d, generator=g).to(dtype).cuda())
            v.append(torch.randn(nb, bs, hkv, d, generator=g).to(dtype).cuda())
    table = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    pool = pa.PagePool(k, v)
    model = PageModel([x.cpu() for x in k], [x.cpu() for x in v], table.cpu(), lens.cpu())
    return pool, model, table, lens, k, v


def _t(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("rows,width,nb,bs,hkv,d,layers,strided", [
    (5, 12, 40, 16, 2, 64, 2, False),       # few pages: runs out
    (37, 9, 700, 8, 1, 128, 1, False),
    (20, 40, 33, 4, 3, 8, 3, True),         # runs out, odd heads, strided caches
    (64, 5, 257, 64, 4, 64, 2, True),
    (3, 600, 1000, 1, 1, 64, 1, False),     # one-token pages, rows of several spans
])
def test_random_serving_sequences(seed, rows, width, nb, bs, hkv, d, layers, strided):
    """Admit, grow, shrink, end, fork and compact at random, with and without a window."""
    pool, model, table, lens, k, v = _setup(rows, width, nb, bs, hkv, d, layers,
                                            strided=strided, seed=seed)
    r = random.Random(1000 * seed + nb)
    cap = width * bs
    for step in range(14):
        kind = r.choice(["resize", "resize", "window", "fork", "compact"])
        if kind == "compact":
            live = pool.compact(table)
            assert int(live) == model.compact()
        elif kind == "fork":
            n = r.randint(1, rows)
            parents = [r.randrange(-1, rows) for _ in range(n)]
            children = [r.randrange(-1, rows) for _ in range(n)]
            pool.fork(table, lens, _t(parents), _t(children))
            model.fork(parents, children)
        else:
            new = [r.choice([0, -1, min(cap, s + 1), min(cap, s + r.randint(1, cap)),
                             max(0, s - r.randint(1, 3 * bs)), r.randint(0, cap)])
                   for s in model.lens]
            win = dict(window=r.choice([1, 3, bs, 2 * bs + 1, cap]), num_sinks=r.choice([0, 1, bs + 1])) \
                if kind == "window" else {}
            pool.resize(table, lens, _t(new), **win)
            model.resize(new, win.get("window"), win.get("num_sinks", 0))
        assert_same(model, pool, table, lens, k, v, f"step {step} {kind}")


def test_rows_that_end_and_begin_in_one_call():
    """Pages freed by a call are there for the same call; the lowest go first."""
    pool, model, table, lens, k, v = _setup(4, 10, 20)
    for new in ([160, 160, 0, 0], [0, 0, 160, 160], [1, 16, 17, 0], [-1, 15, -1, 160]):
        pool.resize(table, lens, _t(new))
        model.resize(new)
        assert_same(model, pool, table, lens, k, v, f"{new}")
    assert model.status == 0


def test_too_few_pages_leave_rows_as_they_were():
    pool, model, table, lens, k, v = _setup(4, 10, 12)
    for new in ([50, 0, 70, 0], [50, 160, 100, 16], [-1, 5, 96, 3]):
        pool.resize(table, lens, _t(new))
        model.resize(new)
        assert_same(model, pool, table, lens, k, v, f"{new}")
    assert model.status == NO_PAGES


def test_growing_from_a_shared_tail_copies_it():
    """A fork cut back into a shared full page, then both rows grow: each gets its own."""
    pool, model, table, lens, k, v = _setup(3, 8, 30)
    steps = [("resize", [64, 0, 0]), ("fork", [0, 0], [1, 2]), ("resize", [-1, 40, -1]),
             ("resize", [41, 41, -1]), ("resize", [40, 40, 70]), ("resize", [50, 50, 71])]
    for s in steps:
        if s[0] == "fork":
            pool.fork(table, lens, _t(s[1]), _t(s[2]))
            model.fork(s[1], s[2])
        else:
            pool.resize(table, lens, _t(s[1]))
            model.resize(s[1])
        assert_same(model, pool, table, lens, k, v, str(s))
    assert model.status == 0


def test_more_pairs_and_rows_than_one_block_holds():
    rows = 2500
    pool, model, table, lens, k, v = _setup(rows, 3, 9000, bs=4, hkv=1, d=8, layers=1)
    new = [(i * 7) % 12 + 1 if i < 1200 else 0 for i in range(rows)]
    pool.resize(table, lens, _t(new))
    model.resize(new)
    assert_same(model, pool, table, lens, k, v, "admit")
    parents, children = [i % 1200 for i in range(1300)], [1200 + i for i in range(1300)]
    children[5] = children[4]                      # named twice
    pool.fork(table, lens, _t(parents), _t(children))
    model.fork(parents, children)
    assert_same(model, pool, table, lens, k, v, "fork")
    assert model.status == BAD_ROW
    new = [0 if i % 3 else min(12, s + 2) for i, s in enumerate(model.lens)]
    pool.resize(table, lens, _t(new))
    model.resize(new)
    assert_same(model, pool, table, lens, k, v, "thin out")
    assert int(pool.compact(table)) == model.compact()
    assert_same(model, pool, table, lens, k, v, "compact")


def test_long_page_lists_go_through_scratch():
    """More pages taken in one call than shared memory lists."""
    pool, model, table, lens, k, v = _setup(3, 3000, 10000, bs=1, hkv=1, d=8, layers=1)
    for new in ([3000, 2999, 100], [0, 3000, 3000]):
        pool.resize(table, lens, _t(new))
        model.resize(new)
        assert_same(model, pool, table, lens, k, v, "long")


def test_bad_input_is_flagged_and_changes_nothing_else():
    pool, model, table, lens, k, v = _setup(4, 6, 30)
    pool.resize(table, lens, _t([40, 50, 0, 0]))
    model.resize([40, 50, 0, 0])
    for new in ([97, -1, -1, -1], [-1, 2 ** 31 - 1, -1, 10]):          # beyond the table
        pool.resize(table, lens, _t(new))
        model.resize(new)
        assert_same(model, pool, table, lens, k, v, "length")
    assert model.status == BAD_SEQLEN
    pairs = ([0, 9, 1, 0], [9, 2, 0, 2])               # no such rows, a child in use, one that works
    pool.fork(table, lens, _t(pairs[0]), _t(pairs[1]))
    model.fork(*pairs)
    assert_same(model, pool, table, lens, k, v, "fork")
    assert model.status == BAD_SEQLEN | BAD_ROW
    table[1, 0], model.table[1][0] = 77, 77            # no page of the pool
    table[1, 1], model.table[1][1] = 29, 29            # a free page
    pool.resize(table, lens, _t([-1, 0, -1, -1]))
    model.resize([-1, 0, -1, -1])
    assert_same(model, pool, table, lens, k, v, "release")
    assert model.status == BAD_SEQLEN | BAD_ROW | BAD_BLOCK


def test_adopt_counts_the_pages_in_use():
    import paged_attention as pa
    from paged_attention import workloads
    lens = torch.tensor([1, 0, 33, 64], dtype=torch.int32, device="cuda")
    w = workloads.build("adopt", 4, 4, 2, 16, torch.float16, lens, 5, 40, seed=1, head_dim=64)
    w.block_table[2] = w.block_table[3]
    pool = pa.PagePool(w.k_cache, w.v_cache)
    pool.adopt(w.block_table, lens)
    model = PageModel([w.k_cache.cpu()], [w.v_cache.cpu()], w.block_table.cpu(), lens.cpu())
    model.adopt()
    assert_same(model, pool, w.block_table, lens, [w.k_cache], [w.v_cache], "adopt")
    w.block_table[0, 0] = 40
    with pytest.raises(ValueError, match="outside the pool"):
        pool.adopt(w.block_table, lens)
    w.block_table[0, 0] = 0
    lens[1] = 5 * 16 + 1
    with pytest.raises(ValueError, match="capacity"):
        pool.adopt(w.block_table, lens)
    with pytest.raises(ValueError):
        pool.adopt(w.block_table, lens.long())


def test_captured_step_replays_on_current_state():
    """resize in a graph beside new_lens = lens + 1, replayed across page borders."""
    pool, model, table, lens, k, v = _setup(6, 20, 200)
    new = [3, 16, 31, 200, 0, 77]
    pool.resize(table, lens, _t(new))
    model.resize(new)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    nxt = torch.zeros_like(lens)
    with torch.cuda.stream(side):
        torch.add(lens, 1, out=nxt)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        torch.add(lens, 1, out=nxt)
        pool.resize(table, lens, nxt, window=40, num_sinks=3)
    for step in range(35):
        graph.replay()
        model.resize([s + 1 for s in model.lens], 40, 3)
        assert_same(model, pool, table, lens, k, v, f"replay {step}")


def test_scratch_does_not_grow_while_capturing():
    import paged_attention as pa
    k = torch.zeros(8, 4, 1, 8, device="cuda", dtype=torch.float16)
    pool = pa.PagePool(k, k.clone())
    table = torch.full((5000, 1), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(5000, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    x = torch.zeros(4, device="cuda")
    with torch.cuda.graph(graph):
        x.add_(1)
        with pytest.raises(RuntimeError, match="before capturing"):
            pool.resize(table, lens, lens)
    graph.replay()
    pool.resize(table, lens, lens)
    assert pool.read_status() == 0


def test_refusals_on_the_device():
    pool, model, table, lens, k, v = _setup(4, 6, 30)
    new = torch.zeros(4, dtype=torch.int32, device="cuda")
    for bad in (lambda: pool.resize(table.long(), lens, new), lambda: pool.resize(table, lens.long(), new),
                lambda: pool.resize(table, lens[:3], new), lambda: pool.resize(table, lens, new[:3]),
                lambda: pool.resize(table.cpu(), lens, new), lambda: pool.resize(table.t(), lens, new),
                lambda: pool.resize(table[:1].expand(4, 6), lens, new),
                lambda: pool.resize(table, lens, new, window=0), lambda: pool.resize(table, lens, new, num_sinks=1),
                lambda: pool.fork(table, lens, new, new[:2]), lambda: pool.compact(table[0])):
        with pytest.raises(ValueError):
            bad()
    assert_same(model, pool, table, lens, k, v, "after refusals")


def test_empty_calls():
    pool, model, table, lens, k, v = _setup(2, 3, 8)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    pool.resize(table[:0], lens[:0], none)
    pool.fork(table, lens, none, none)
    assert int(pool.compact(table)) == 0
    assert int(pool.compact(table[:0])) == 0
    assert_same(model, pool, table, lens, k, v, "empty")


@pytest.mark.parametrize("nb", [900, 1400, 4000])
def test_tails_that_all_users_leave_are_free_only_after_the_call(nb):
    """Shared last pages among the first 1024 rows lose their last user while later rows
    still take pages: the numbering of the free pages must not move meanwhile."""
    rows, bs = 2100, 4
    pool, model, table, lens, k, v = _setup(rows, 3, nb, bs, 1, 8, 1, seed=nb)
    r = random.Random(nb)
    low = r.sample(range(0, nb // 4), 60)
    start = torch.zeros(rows, dtype=torch.int32)
    for i, page in enumerate(low):                  # two to four users each, also across 1024
        for row in r.sample(range(i * 30, i * 30 + 30), r.randint(2, 3)) + [1024 + i]:
            table[row, 0] = page
            start[row] = 2
    lens.copy_(start)
    model.table, model.lens = table.tolist(), lens.tolist()
    pool.adopt(table, lens)
    model.adopt()
    new = [r.choice([-1, 3, 4, 5, 9]) if s else r.choice([-1, 0, 1, 5]) for s in start.tolist()]
    pool.resize(table, lens, _t(new))
    model.resize(new)
    assert_same(model, pool, table, lens, k, v, "grown")
    new = [r.choice([-1, 0, 12]) for _ in range(rows)]
    pool.resize(table, lens, _t(new))
    model.resize(new)
    assert_same(model, pool, table, lens, k, v, "again")


@pytest.mark.parametrize("sinks", [2 ** 31 - 1, 2 ** 31 - 16, 2 ** 40])
def test_first_tokens_without_end_are_kept(sinks):
    pool, model, table, lens, k, v = _setup(2, 8, 20)
    for new in ([128, 70], [128, 100]):
        pool.resize(table, lens, _t(new), window=16, num_sinks=sinks)
        model.resize(new, 16, sinks)
        assert_same(model, pool, table, lens, k, v, f"{new}")
    assert model.refs.count(1) == 15
