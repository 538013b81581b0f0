"""GPU tests of the windowed operators in a pool whose element offsets pass 32 bits."""
import pytest
import torch

from window_helpers import PoisonedCache, assert_matches, reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", params=[16, 12])
def far(request):
    """A small cache's pages moved behind element 2^32 of a large pool."""
    bs = request.param
    window, sinks, qs, lens = 150, 4, [70, 1, 300], [700, 33, 300]
    c = PoisonedCache(lens, qs, 8, 128, bs, torch.float16, window, sinks, 5)
    pages = (2 ** 32 + 2 ** 28) // (bs * 8 * 128)
    k = torch.empty(pages, bs, 8, 128, dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    n = c.k.shape[0]
    k[-n:], v[-n:] = c.k, c.v
    table = torch.where(c.table >= 0, c.table + (pages - n), c.table)
    yield bs, window, sinks, qs, c, k, v, table
    del k, v
    torch.cuda.empty_cache()


def test_attention_behind_element_2_to_32(far):
    import paged_attention as pa
    bs, window, sinks, qs, c, k, v, table = far
    st = torch.tensor([0, 70, 71, 371], dtype=torch.int32, device="cuda")
    q = torch.randn(371, 16, 128, device="cuda").half()
    o = pa.paged_prompt_attention(q, k, v, table, st, c.lens, bs, window=window, num_sinks=sinks)
    want, _, tol = reference(q, c.k, c.v, c.table, c.lens, bs, window, sinks, st)
    vmax = c.v[~c.v.isnan()].abs().max().double().item()
    assert_matches(o, want, tol + 2.0 ** -11 * vmax, "prompt")
    last = q[[69, 70, 370]].contiguous()
    o = pa.paged_attention(last, k, v, table, c.lens, bs, window=window, num_sinks=sinks)
    want, _, tol = reference(last, c.k, c.v, c.table, c.lens, bs, window, sinks)
    assert_matches(o, want, tol, "decode")


def test_pages_behind_element_2_to_32(far):
    import paged_attention as pa
    bs, window, sinks, qs, c, k, v, table = far
    pool = pa.PagePool(k, v)
    table = torch.cat([table, torch.full_like(table[:1], -1)])
    lens = torch.cat([c.lens, torch.zeros_like(c.lens[:1])])
    pool.adopt(table, lens)
    live = int((pool.refs > 0).sum())
    before = [x[table[0, 650 // bs].long()].clone() for x in (k, v)]
    tail = [x[table[0, 700 // bs].long(), : 700 % bs].clone() for x in (k, v)]
    # the pages below 2^32 are taken up to the last ones, so that the copy's page is high too
    pool.refs[: k.shape[0] - 64] += 1
    pool._pool.free_words[: (k.shape[0] - 64) // 32].zero_()
    pool.fork(table, lens, torch.tensor([0], device="cuda"), torch.tensor([3], device="cuda"))
    assert pool.read_status() == 0 and int(lens[3]) == 700
    for x, t in zip((k, v), tail):
        assert torch.equal(x[table[3, 700 // bs].long(), : 700 % bs], t)
    pool.adopt(table, lens)
    assert int(pool.compact(table)) == live + 1
    assert int(table.max()) == live
    for x, a, t in zip((k, v), before, tail):
        for row in (0, 3):
            assert torch.equal(x[table[row, 650 // bs].long()].view(torch.int16), a.view(torch.int16))
            assert torch.equal(x[table[row, 700 // bs].long(), : 700 % bs], t)


def test_rows_that_ask_for_more_than_2_to_31_pages():
    """Sums and lengths at the end of int32: refused for lack of pages, each by itself."""
    import paged_attention as pa
    rows, width = 1100, 2 ** 21
    k = torch.zeros(64, 1, 1, 8, dtype=torch.float16, device="cuda")
    pool = pa.PagePool(k, torch.zeros_like(k))
    table = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    new = torch.full_like(lens, width)
    new[:2] = 20
    pool.resize(table, lens, new)
    assert lens.tolist() == [20, 20] + [0] * (rows - 2)
    assert pool.read_status() == pa._native.PA_STATUS_NO_PAGES
    assert table[:2, :20].flatten().tolist() == list(range(40))
    assert int((table >= 0).sum()) == 40 and int(pool.refs.sum()) == 40
    # one row's length just below 2^31 tokens, in pages of 1024
    k = torch.zeros(64, 1024, 1, 8, dtype=torch.float16, device="cuda")
    pool = pa.PagePool(k, torch.zeros_like(k))
    table = torch.full((3, width), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(3, dtype=torch.int32, device="cuda")
    new = torch.tensor([5, 2 ** 31 - 1, 0], dtype=torch.int32, device="cuda")
    pool.resize(table, lens, new)
    assert lens.tolist() == [5, 0, 0]
    assert pool.read_status() == pa._native.PA_STATUS_NO_PAGES
