"""GPU tests of windowed decode (``paged_attention(..., window=, num_sinks=)``)
against the definition in 64 bits, over caches whose invisible slots are NaN and
whose invisible pages are not there."""
import ctypes

import pytest
import torch

from window_helpers import PoisonedCache, assert_lse, assert_matches, reference

pytestmark = pytest.mark.gpu


def _lens(window, sinks, bs):
    """Lengths where the window, the sinks and the pages meet."""
    base = [0, 1, 2, bs - 1, bs, bs + 1, window - 1, window, window + 1, window + sinks - 1,
            window + sinks, window + sinks + 1, window + bs, window + sinks + 2 * bs + 1,
            window + 16, window + 32, window + 33, 3 * window + 5, 1500]
    return sorted({max(0, min(1500, x)) for x in base})


def _run(lens, hq, hkv, d, bs, dtype, window, sinks, seed, **kw):
    import paged_attention as pa
    c = PoisonedCache(lens, [1] * len(lens), hkv, d, bs, dtype, window, sinks, seed)
    g = torch.Generator().manual_seed(seed + 1)
    q = torch.randn(len(lens), hq, d, generator=g).to(dtype).cuda()
    ws = pa.DecodeWorkspace("cuda")
    o, lse = pa.paged_attention(q, c.k, c.v, c.table, c.lens, bs, window=window,
                                num_sinks=sinks, return_lse=True, workspace=ws, **kw)
    torch.cuda.synchronize()
    assert ws.read_status() == 0
    return c, q, o, lse


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (7, 1), (64, 4), (100, 40), (512, 0),
                                          (4000, 4)])
@pytest.mark.parametrize("hkv,g,d,bs", [(2, 4, 128, 16), (3, 1, 64, 32), (2, 8, 128, 16),
                                        (1, 3, 128, 8), (2, 2, 256, 16), (2, 12, 64, 64),
                                        (1, 2, 32, 16), (2, 1, 64, 1), (1, 5, 128, 24),
                                        (2, 1, 128, 12)])
def test_window_decode(dtype, window, sinks, hkv, g, d, bs):
    lens = _lens(window, sinks, bs)
    c, q, o, lse = _run(lens, hkv * g, hkv, d, bs, dtype, window, sinks, seed=d + bs + g)
    want, wl, tol = reference(q, c.k, c.v, c.table, c.lens, bs, window, sinks)
    what = f"{dtype} w{window} s{sinks} d{d} bs{bs} g{g}"
    assert_matches(o, want, tol, what)
    assert_lse(lse, wl, d, what)


@pytest.mark.parametrize("length", [1, 40, 300, 5000])
@pytest.mark.parametrize("hkv,g,d", [(8, 4, 128), (32, 1, 128), (4, 8, 64)])
def test_window_decode_scalar_length(length, hkv, g, d):
    """One length for every row (an int), and a single long stream (merge pass)."""
    import paged_attention as pa
    window, sinks, bs = 1024, 4, 16
    for batch in (1, 3):
        lens = [length] * batch
        c = PoisonedCache(lens, [1] * batch, hkv, d, bs, torch.bfloat16, window, sinks, 11)
        q = torch.randn(batch, hkv * g, d, device="cuda").bfloat16()
        o, lse = pa.paged_attention(q, c.k, c.v, c.table, length, bs, window=window,
                                    num_sinks=sinks, return_lse=True)
        o2, lse2 = pa.paged_attention(q, c.k, c.v, c.table, c.lens, bs, window=window,
                                      num_sinks=sinks, return_lse=True)
        want, wl, tol = reference(q, c.k, c.v, c.table, lens, bs, window, sinks)
        assert_matches(o, want, tol, f"scalar {length}")
        assert_lse(lse, wl, d, f"scalar {length}")
        assert torch.equal(o, o2) and torch.equal(lse, lse2)


def test_window_that_covers_everything_is_full_attention():
    import paged_attention as pa
    from paged_attention import workloads
    lens = torch.tensor([1, 17, 300, 999, 64], dtype=torch.int32, device="cuda")
    w = workloads.build("wide", 5, 16, 4, 16, torch.bfloat16, lens, 63, 400, seed=3)
    full = pa.paged_attention(w.q, w.k_cache, w.v_cache, w.block_table, lens, 16)
    for window in (999, 1000, 10 ** 6, 2 ** 40):
        got = pa.paged_attention(w.q, w.k_cache, w.v_cache, w.block_table, lens, 16,
                                 window=window, num_sinks=4)
        # the schedules may split rows elsewhere: one rounding of the output apart
        assert_matches(got, full.double().cpu(), 2 * 2.0 ** -8 * full.double().cpu().abs() + 1e-5,
                       f"window {window}")


@pytest.mark.parametrize("batch", [1024, 1025, 2100])
def test_window_decode_beyond_the_per_row_limit(batch):
    """More rows than one launch's schedule holds."""
    lens = [(i * 37) % 90 for i in range(batch)]
    c, q, o, lse = _run(lens, 2, 1, 64, 16, torch.float16, 20, 3, seed=5)
    want, wl, tol = reference(q, c.k, c.v, c.table, c.lens, 16, 20, 3)
    assert_matches(o, want, tol, f"batch {batch}")
    assert_lse(lse, wl, 64, f"batch {batch}")


def test_window_decode_strided_inputs_and_out():
    """Caches that are slices of a joint [pages, 2, slots, heads, D] buffer, a strided q, a given out."""
    import paged_attention as pa
    lens, window, sinks, bs, hkv, d = [5, 700, 90], 100, 4, 16, 2, 128
    c = PoisonedCache(lens, [1] * 3, hkv, d, bs, torch.float16, window, sinks, 7)
    kv = torch.stack([c.k, c.v], 1)
    qbig = torch.randn(3, 5, 2 * hkv, d, device="cuda").half()
    q = qbig[:, 2]
    out = torch.full((4, 2 * hkv, d), 7.0, device="cuda").half()
    got = pa.paged_attention(q, kv[:, 0], kv[:, 1], c.table, c.lens, bs, window=window,
                             num_sinks=sinks, out=out[:3])
    want, _, tol = reference(q, c.k, c.v, c.table, lens, bs, window, sinks)
    assert got.data_ptr() == out.data_ptr()
    assert_matches(got, want, tol, "strided")
    assert (out[3] == 7).all()


def test_window_graph_runner_follows_lengths():
    import paged_attention as pa
    window, sinks, bs, hkv, g, d, b = 50, 4, 16, 2, 4, 128, 4
    runner = pa.PagedAttnGraphRunner(b, hkv * g, d, 16, bs, 64, dtype=torch.bfloat16,
                                     num_kv_heads=hkv, dynamic_seq_lens=True, max_seq_len=640,
                                     window=window, num_sinks=sinks)
    for k, lens in enumerate(([1, 40, 300, 640], [0, 55, 54, 90], [640, 640, 1, 2])):
        c = PoisonedCache(lens, [1] * b, hkv, d, bs, torch.bfloat16, window, sinks, k, width=40)
        q = torch.randn(b, hkv * g, d, device="cuda").bfloat16()
        pool = torch.full((64, bs, hkv, d), float("nan"), device="cuda").bfloat16()
        kk, vv = pool.clone(), pool.clone()
        kk[: c.k.shape[0]], vv[: c.v.shape[0]] = c.k, c.v
        out = runner.run(q, kk, vv, c.table, copy_kv=True, seq_lens=c.lens)
        want, _, tol = reference(q, c.k, c.v, c.table, lens, bs, window, sinks)
        assert_matches(out, want, tol, f"graph {lens}")


def test_window_decode_on_another_stream():
    lens = [2000] * 6
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        c, q, o, lse = _run(lens, 8, 2, 128, 16, torch.bfloat16, 300, 4, seed=9)
    want, wl, tol = reference(q, c.k, c.v, c.table, c.lens, 16, 300, 4)
    assert_matches(o, want, tol, "side stream")


@pytest.mark.parametrize("d,variants", [(128, (1, 2, 3, 4, 5, 10)), (64, (3, 5, 8)), (256, (6, 7, 9))])
@pytest.mark.parametrize("g", [1, 4, 8])
def test_window_decode_every_variant(d, variants, g):
    lens = [1, 30, 31, 140, 900, 0, 333]
    for v in variants:
        c, q, o, lse = _run(lens, 2 * g, 2, d, 16, torch.bfloat16, 100, 20, seed=v, kernel_variant=v)
        want, wl, tol = reference(q, c.k, c.v, c.table, c.lens, 16, 100, 20)
        assert_matches(o, want, tol, f"variant {v}")
        assert_lse(lse, wl, d, f"variant {v}")


def test_window_decode_flags_bad_page_and_length():
    """A visible page outside the pool and a length beyond the table are flagged, not fatal;
    an invisible page may be anything."""
    import paged_attention as pa
    from paged_attention import _native
    c = PoisonedCache([200, 200], [1, 1], 1, 64, 16, torch.float16, 50, 4, 3)
    q = torch.randn(2, 1, 64, device="cuda").half()
    ws = pa.DecodeWorkspace("cuda")
    c.table[0, 5] = 10 ** 6                      # tokens 80..95: not visible
    pa.paged_attention(q, c.k, c.v, c.table, c.lens, 16, window=50, num_sinks=4, workspace=ws)
    assert ws.read_status() == 0
    c.table[0, 11] = 10 ** 6                     # tokens 176..191: visible
    pa.paged_attention(q, c.k, c.v, c.table, c.lens, 16, window=50, num_sinks=4, workspace=ws)
    assert ws.read_status() == _native.PA_STATUS_BAD_BLOCK
    ws.reset()
    c.lens[1] = 16 * 13 + 1
    pa.paged_attention(q, c.k, c.v, c.table, c.lens, 16, window=50, num_sinks=4, workspace=ws)
    assert ws.read_status() & _native.PA_STATUS_BAD_SEQLEN


def test_window_decode_through_ctypes_with_its_own_workspace():
    import paged_attention as pa
    from paged_attention import _native
    lens, window, sinks, bs, hkv, d = [900, 3, 0], 128, 4, 16, 2, 128
    c = PoisonedCache(lens, [1] * 3, hkv, d, bs, torch.bfloat16, window, sinks, 1)
    q = torch.randn(3, 4 * hkv, d, device="cuda").bfloat16()
    out = torch.empty_like(q)
    p = pa.decode_params(q, c.k, c.v, c.table, c.lens, bs, out=out)
    lib = _native.lib()
    nb, nc = ctypes.c_size_t(), ctypes.c_size_t()
    assert lib.pa_window_decode_workspace(ctypes.byref(p), window, sinks, ctypes.byref(nb),
                                          ctypes.byref(nc)) == 0
    buf = torch.empty(max(16, nb.value), dtype=torch.uint8, device="cuda")
    cnt = torch.zeros(max(1, nc.value), dtype=torch.int32, device="cuda")
    p.workspace, p.workspace_bytes = buf.data_ptr(), nb.value
    p.counters, p.counter_count = cnt.data_ptr(), nc.value
    stream = torch.cuda.current_stream().cuda_stream
    for _ in range(2):
        assert lib.pa_window_decode(ctypes.byref(p), window, sinks, stream) == 0
        want, _, tol = reference(q, c.k, c.v, c.table, lens, bs, window, sinks)
        assert_matches(out, want, tol, "ctypes")
        out.zero_()
        assert int(cnt.abs().sum()) == 0


@pytest.mark.parametrize("d,bs", [(32, 16), (64, 5), (128, 5), (128, 16), (256, 32)])
@pytest.mark.parametrize("s", [1, 40, 700])
def test_nan_in_visible_places_shows(d, bs, s):
    """A visible key's NaN makes its KV head's rows NaN, a value's its dimension, also where
    a split holds no other token; the other head's rows keep their bits."""
    import paged_attention as pa
    g = torch.Generator().manual_seed(s + d)
    pages = -(-s // bs)
    k, v = (torch.randn(pages, bs, 2, d, generator=g).half().cuda() for _ in range(2))
    q = torch.randn(3, 4, d, generator=g).half().cuda()
    table = torch.arange(pages, dtype=torch.int32, device="cuda").repeat(3, 1)
    lens = torch.full((3,), s, dtype=torch.int32, device="cuda")

    def run():
        return pa.paged_attention(q, k, v, table, lens, bs, window=350, num_sinks=2)
    clean = run()
    assert clean.isfinite().all()
    for t in sorted({0, s // 2, s - 1} if s < 700 else {0, 350, 500, 699}):
        for x, dims in ((k, slice(None)), (v, slice(5, 6))):
            kept = x[t // bs, t % bs, 0, 5].clone()
            x[t // bs, t % bs, 0, 5] = float("nan")
            o = run()
            x[t // bs, t % bs, 0, 5] = kept
            assert o[:, :2, dims].isnan().all(), f"token {t}"
            o[:, :2, dims] = clean[:, :2, dims]
            assert torch.equal(o, clean)


def _odd_numbers_case(d, bs, hkv, g, batch, s, seed):
    gen = torch.Generator().manual_seed(seed)
    pages = -(-s // bs)
    k, v = (torch.randn(pages, bs, hkv, d, generator=gen).half().cuda() for _ in range(2))
    q = (torch.rand(batch, hkv * g, d, generator=gen) + 0.01).half().cuda()
    table = torch.arange(pages, dtype=torch.int32, device="cuda").repeat(batch, 1)
    return q, k, v, table, torch.full((batch,), s, dtype=torch.int32, device="cuda")


# (one row and many, groups and full heads, rows merged in every place where pieces meet)
ODD_SHAPES = [(128, 16, 8, 4, 1), (128, 16, 32, 1, 1), (128, 16, 2, 4, 3), (128, 16, 2, 8, 2), (128, 32, 4, 3, 40),
              (64, 16, 2, 4, 1), (64, 32, 3, 1, 30), (256, 32, 2, 2, 1), (256, 16, 1, 8, 9),
              # on the CUDA cores
              (32, 16, 2, 4, 1), (32, 8, 3, 1, 9), (64, 5, 2, 2, 3), (128, 1, 1, 4, 2), (256, 12, 2, 1, 1)]


@pytest.mark.parametrize("d,bs,hkv,g,batch", ODD_SHAPES)
@pytest.mark.parametrize("s,window,sinks", [(1, 1, 0), (3000, 1024, 1), (700, 350, 2), (900, 1, 1)])
def test_nan_and_infinite_scores_show_in_output_and_lse(d, bs, hkv, g, batch, s, window, sinks):
    """A NaN query, or a visible key that scores NaN or +infinity, makes its rows NaN, their
    LSE too, also where it is the only token of a tile; the others keep their bits."""
    import paged_attention as pa
    q, k, v, table, lens = _odd_numbers_case(d, bs, hkv, g, batch, s, seed=s + d + g)

    def run(q):
        return pa.paged_attention(q, k, v, table, lens, bs, window=window, num_sinks=sinks, return_lse=True)
    clean, clean_lse = run(q)
    assert clean.isfinite().all() and clean_lse.isfinite().all()

    def check(got, rows, heads, what):
        o, lse = got
        assert o[rows, heads].isnan().all(), f"{what}: O"
        assert lse[rows, heads].isnan().all(), f"{what}: LSE"
        o[rows, heads], lse[rows, heads] = clean[rows, heads], clean_lse[rows, heads]
        assert torch.equal(o, clean) and torch.equal(lse, clean_lse), f"{what}: other rows"
    bad = q.clone()
    bad[batch // 2, hkv * g - 1, 3] = float("nan")
    check(run(bad), batch // 2, hkv * g - 1, "query")
    every = slice(None)
    low = max(0, s - window)
    for t in sorted({0, low, (low + s) // 2, s - 1} - (set() if sinks or not low else {0})):
        for value in (float("nan"), float("inf")):
            kept = k[t // bs, t % bs, hkv - 1, 5].clone()
            k[t // bs, t % bs, hkv - 1, 5] = value
            got = run(q)
            k[t // bs, t % bs, hkv - 1, 5] = kept
            check(got, every, slice((hkv - 1) * g, hkv * g), f"key {t} {value}")


@pytest.mark.parametrize("d,bs,hkv,g,batch", ODD_SHAPES)
@pytest.mark.parametrize("s,window,sinks", [(1, 1, 0), (3000, 1024, 1), (700, 350, 2)])
def test_scores_of_minus_infinity_weigh_nothing(d, bs, hkv, g, batch, s, window, sinks):
    """Visible keys that score -infinity: some, whole tiles of them, all (as if nothing were seen)."""
    import paged_attention as pa
    q, k, v, table, lens = _odd_numbers_case(d, bs, hkv, g, batch, s, seed=s + d)
    seen = torch.tensor([t for t in range(s) if t < sinks or t >= s - window])
    for dead in (seen[:1], seen[: len(seen) // 2], seen[len(seen) // 3:], seen):
        kk = k.clone()
        kk[dead.cuda() // bs, dead.cuda() % bs, :, 5] = float("-inf")
        o, lse = pa.paged_attention(q, kk, v, table, lens, bs, window=window, num_sinks=sinks, return_lse=True)
        left = torch.tensor(sorted(set(seen.tolist()) - set(dead.tolist())), dtype=torch.long)
        if not len(left):
            assert (o == 0).all() and (lse == -1e30).all()
            continue
        # the same rows over the tokens that are left, in 64 bits; tolerances as in the definition's helper
        k2, v2 = (x.cpu()[left // bs, left % bs].double().repeat_interleave(g, 1) for x in (k, v))
        sc = torch.einsum("bhd,thd->bht", q.cpu().double(), k2) * d ** -0.5
        big = (torch.einsum("bhd,thd->bht", q.cpu().double(), k2.abs()) * d ** -0.5).amax(-1, keepdim=True)
        want = torch.einsum("bht,thd->bhd", torch.softmax(sc, -1), v2)
        tol = (2 * d * 2.0 ** -24 * big + 2.0 ** -16) * v2.abs().max() + 2.0 ** -11 * want.abs()
        assert_matches(o, want, tol, f"{len(dead)} of {len(seen)} at -infinity")
        assert_lse(lse, torch.logsumexp(sc, -1), d, f"{len(dead)} of {len(seen)} at -infinity")


def _misplaced(q):
    """The same queries [N, H, D] off their 16 bytes, and a single one with an odd stride."""
    flat = torch.zeros(q.numel() + 1, dtype=q.dtype, device=q.device)
    flat[1:] = q.reshape(-1)
    yield flat[1:].view(q.shape), slice(None)
    odd = torch.zeros(q[0].numel() + 1, dtype=q.dtype, device=q.device)
    odd[:-1] = q[0].reshape(-1)
    yield odd.as_strided((1, *q.shape[1:]), (q[0].numel() + 1, q.shape[2], 1)), slice(0, 1)


@pytest.mark.parametrize("window,sinks", [(100, 4), (None, 0)])
@pytest.mark.parametrize("d,bs", [(128, 16), (32, 16), (64, 5)])
def test_queries_off_their_alignment_are_copied(d, bs, window, sinks):
    import paged_attention as pa
    lens = [150, 3, 40]
    c = PoisonedCache(lens, [1] * 3, 2, d, bs, torch.float16, window or 10 ** 9, sinks, 5)
    q = torch.randn(3, 6, d, device="cuda").half()
    want = pa.paged_attention(q, c.k, c.v, c.table, c.lens, bs, window=window, num_sinks=sinks)
    starts = torch.arange(4, dtype=torch.int32, device="cuda")
    pwant = pa.paged_prompt_attention(q, c.k, c.v, c.table, starts, c.lens, bs, window=window,
                                      num_sinks=sinks, num_splits=1)
    for x, rows in _misplaced(q):
        n = len(x)
        got = pa.paged_attention(x, c.k, c.v, c.table[rows], c.lens[rows], bs, window=window, num_sinks=sinks)
        # (one row alone may be split elsewhere: a rounding of the output apart)
        assert_matches(got, want[rows].double().cpu(), (0 if n == 3 else 2 * 2.0 ** -11)
                       * want[rows].double().cpu().abs() + (0 if n == 3 else 1e-5), "decode")
        got = pa.paged_prompt_attention(x, c.k, c.v, c.table[rows], starts[: n + 1], c.lens[rows], bs,
                                        window=window, num_sinks=sinks, num_splits=1)
        assert torch.equal(got, pwant[rows])


def test_tangents_are_refused():
    """Forward-mode derivatives through the windowed calls and prompt attention do not exist."""
    import paged_attention as pa
    import torch.autograd.forward_ad as fw
    c = PoisonedCache([50, 7], [1, 1], 2, 64, 16, torch.float16, 20, 2, 5)
    q = torch.randn(2, 4, 64, device="cuda").half()
    starts = torch.arange(3, dtype=torch.int32, device="cuda")

    def calls(q, k, v):
        return (lambda: pa.paged_attention(q, k, v, c.table, c.lens, 16, window=20, num_sinks=2),
                lambda: pa.paged_prompt_attention(q, k, v, c.table, starts, c.lens, 16, window=20, num_sinks=2))
    want = [f() for f in calls(q, c.k, c.v)]
    with fw.dual_level():
        for i in range(3):
            args = [q, c.k, c.v]
            args[i] = fw.make_dual(args[i], torch.ones_like(args[i]))
            for f, w in zip(calls(*args), want):
                with pytest.raises(RuntimeError, match="inference-only"):
                    f()
                with torch.inference_mode():          # asks for no derivative
                    assert torch.equal(f(), w)
        for f, w in zip(calls(q, c.k, c.v), want):
            assert torch.equal(f(), w)


@pytest.mark.parametrize("kw", [{}, dict(window=20, num_sinks=2)])
def test_out_and_workspace_of_another_device_are_refused(kw):
    import paged_attention as pa
    c = PoisonedCache([50, 7], [1, 1], 2, 64, 16, torch.float16, 20 if kw else 10 ** 9, 2 if kw else 0, 5)
    q = torch.randn(2, 4, 64, device="cuda").half()
    starts = torch.arange(3, dtype=torch.int32, device="cuda")
    for bad in (dict(out=torch.empty(2, 4, 64).half()), dict(workspace=pa.DecodeWorkspace("cpu"))):
        with pytest.raises(ValueError, match="device"):
            pa.paged_attention(q, c.k, c.v, c.table, c.lens, 16, **kw, **bad)
        with pytest.raises(ValueError, match="device"):
            pa.paged_prompt_attention(q, c.k, c.v, c.table, starts, c.lens, 16, **kw, **bad)


def test_out_in_pinned_host_memory():
    import paged_attention as pa
    c = PoisonedCache([50, 7], [1, 1], 2, 64, 16, torch.float16, 20, 2, 5)
    q = torch.randn(2, 4, 64, device="cuda").half()
    want = pa.paged_attention(q, c.k, c.v, c.table, c.lens, 16, window=20, num_sinks=2)
    out = torch.empty(2, 4, 64).half().pin_memory()
    pa.paged_attention(q, c.k, c.v, c.table, c.lens, 16, window=20, num_sinks=2, out=out)
    torch.cuda.synchronize()
    assert torch.equal(out, want.cpu())


def test_caches_without_heads_are_refused():
    import paged_attention as pa
    k = torch.empty(4, 16, 0, 64, device="cuda").half()
    q = torch.zeros(2, 4, 64, device="cuda").half()
    i = torch.zeros(3, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="multiple of Hkv"):
        pa.paged_attention(q, k, k, i.view(3, 1)[:2], i[:2], 16, window=4)
    with pytest.raises(ValueError, match="multiple of Hkv"):
        pa.paged_prompt_attention(q, k, k, i.view(3, 1)[:2], i, i[:2], 16)


@pytest.mark.parametrize("hkv,g,d", [(1, 4, 64), (2, 1, 128), (1, 8, 256), (1, 3, 32)])
@pytest.mark.parametrize("lens,window,sinks", [([5, 700, 0, 1024], 100, 4),
                                               ([2 ** 31 - 65, 2 ** 30 + 3, 1], 130, 3)])
def test_window_decode_over_a_table_of_two_to_the_31_tokens(hkv, g, d, lens, window, sinks):
    """Tables wider than int32 counts tokens, nearly all of it pages that are not there; rows
    at both ends of them."""
    import paged_attention as pa
    from paged_attention import _native
    bs, width = 1024, 2 ** 21
    c = PoisonedCache(lens, [1] * len(lens), hkv, d, bs, torch.bfloat16, window, sinks, d, width=width)
    q = torch.randn(len(lens), hkv * g, d, device="cuda").bfloat16()
    ws = pa.DecodeWorkspace("cuda")

    def run(n, batch):
        return pa.paged_attention(q[:batch], c.k, c.v, c.table[:batch], n, bs, window=window, num_sinks=sinks,
                                  return_lse=True, workspace=ws)
    want, wl, tol = reference(q, c.k, c.v, c.table, lens, bs, window, sinks)
    o, lse = run(c.lens, len(lens))
    assert ws.read_status() == 0
    assert_matches(o, want, tol, f"{lens}")
    assert_lse(lse, wl, d, f"{lens}")
    o, lse = run(lens[0], 1)
    assert_matches(o, want[:1], tol[:1], f"{lens[0]}")
    assert_lse(lse, wl[:1], d, f"{lens[0]}")
    assert ws.read_status() == 0
    c.lens[1] = 2 ** 31 - 1                    # longer than a length can be: cut and flagged
    c.table[1, -1] = c.table[0, 0] if lens[0] < bs else c.table[0, -1]
    o, lse = run(c.lens, len(lens))
    assert ws.read_status() & _native.PA_STATUS_BAD_SEQLEN
    keep = [0] + list(range(2, len(lens)))
    assert_matches(o[keep], want[keep], tol[keep], "the other rows")
