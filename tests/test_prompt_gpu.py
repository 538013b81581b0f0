"""GPU tests of prompt attention (``paged_prompt_attention``) against the definition in
64 bits, over caches whose invisible slots are NaN and whose invisible pages are not
there."""
import ctypes

import pytest
import torch

from window_helpers import PoisonedCache, assert_lse, assert_matches, reference

pytestmark = pytest.mark.gpu


def _starts(qs):
    out = [0]
    for n in qs:
        out.append(out[-1] + n)
    return out


def _tolerance(q, tol, want_abs_v):
    """The definition's tolerance, with probabilities rounded once to the 16-bit type
    (half a step, relative) before the product with V: at most that times max|v|."""
    return tol + torch.finfo(q.dtype).eps / 2 * want_abs_v


def _run(qs, lens, hq, hkv, d, bs, dtype, window, sinks, seed, pad=0, **kw):
    import paged_attention as pa
    full = window is None
    win = 10 ** 9 if full else window
    c = PoisonedCache(lens, qs, hkv, d, bs, dtype, win, sinks, seed)
    g = torch.Generator().manual_seed(seed + 1)
    starts = _starts(qs)
    q = torch.randn(starts[-1] + pad, hq, d, generator=g).to(dtype).cuda()
    ws = pa.DecodeWorkspace("cuda")
    out = torch.full_like(q, 7.0)
    st = torch.tensor(starts, dtype=torch.int32, device="cuda")
    o, lse = pa.paged_prompt_attention(q, c.k, c.v, c.table, st, c.lens, bs, window=window,
                                       num_sinks=sinks, return_lse=True, workspace=ws, out=out,
                                       **kw)
    torch.cuda.synchronize()
    assert ws.read_status() == 0
    want, wl, tol = reference(q, c.k, c.v, c.table, lens, bs, win, sinks, starts)
    n = starts[-1]
    vmax = c.v[~c.v.isnan()].abs().max().double().item() if (~c.v.isnan()).any() else 0.0
    what = f"{dtype} q{qs} s{lens} w{window} k{sinks} d{d} bs{bs} hq{hq}/{hkv} {kw}"
    assert_matches(o[:n], want[:n], _tolerance(q, tol, vmax)[:n], what)
    assert_lse(lse[:n], wl[:n], d, what)
    assert (o[n:] == 7).all(), "rows behind the last sequence"
    return c, q, st, o, lse


SHAPES = [(2, 4, 128, 16), (3, 1, 64, 32), (1, 8, 128, 16), (1, 3, 128, 8), (1, 2, 256, 16),
          (2, 5, 64, 64), (1, 2, 32, 16), (1, 2, 64, 1), (1, 4, 128, 24), (1, 2, 256, 128),
          (1, 1, 128, 12), (1, 16, 64, 8), (1, 2, 128, 256)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (1, 3), (37, 5), (128, 4), (200, 140)])
@pytest.mark.parametrize("hkv,g,d,bs", SHAPES)
def test_prompt_small(dtype, window, sinks, hkv, g, d, bs):
    """Chunks of 0 to 100 tokens at the start, in the middle and at the end of sequences."""
    qs = [1, 0, 5, 33, 17, 100, 0, 2]
    lens = [1, 9, 300, 33, 146, 129, 0, 513]
    _run(qs, lens, hkv * g, hkv, d, bs, dtype, window, sinks, seed=d + bs + g, pad=3)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hkv,g,d,bs", [(1, 4, 128, 16), (2, 1, 64, 32), (1, 2, 256, 16)])
@pytest.mark.parametrize("qs,lens,window,sinks", [
    ([300], [300], None, 0),
    ([257, 128], [700, 128], 130, 4),
    ([256, 64, 65], [256, 1000, 1025], 256, 1),
    ([600], [900], 64, 300),
])
def test_prompt_several_tiles(dtype, hkv, g, d, bs, qs, lens, window, sinks):
    _run(qs, lens, hkv * g, hkv, d, bs, dtype, window, sinks, seed=sum(qs))


@pytest.mark.parametrize("splits", [1, 2, 3, 7, 40])
@pytest.mark.parametrize("window,sinks", [(None, 0), (500, 4)])
def test_prompt_splits(splits, window, sinks):
    """The keys in parts that a second kernel joins; more parts than tiles too."""
    _run([7, 1, 0, 40], [1500, 1, 30, 640], 8, 2, 128, 16, torch.bfloat16, window, sinks,
         seed=splits, pad=2, num_splits=splits)
    _run([3, 20], [999, 2000], 4, 4, 64, 16, torch.float16, window, sinks, seed=splits,
         num_splits=splits)
    _run([3], [400], 4, 2, 256, 32, torch.float16, window, sinks, seed=splits, num_splits=splits)


def test_prompt_rows_before_the_sequence_see_nothing():
    """A chunk longer than its sequence: its first rows sit before position 0."""
    for d, bs in ((128, 16), (32, 16)):
        c, q, st, o, lse = _run([40, 9], [25, 0], 4, 2, d, bs, torch.float16, 8, 2, seed=4)
        assert (o[:15] == 0).all() and (lse[:15] == -1e30).all()
        assert (o[40:49] == 0).all() and (lse[40:49] == -1e30).all()


@pytest.mark.parametrize("hkv,g,d", [(4, 4, 128), (8, 1, 128), (8, 4, 64), (4, 4, 32), (2, 4, 256)])
def test_prompt_rows_that_see_nothing_are_zero_over_large_queries(hkv, g, d):
    """Whole row tiles without a visible token: what is staged of their queries, which come
    from memory late, must not end up in the output."""
    import paged_attention as pa
    n, b = 1024, 6
    k = torch.full((4, 16, hkv, d), 3.0, device="cuda").half()
    table = torch.full((b, 4), -1, dtype=torch.int32, device="cuda")
    starts = torch.arange(0, n * b + 1, n, dtype=torch.int32, device="cuda")
    lens = torch.zeros(b, dtype=torch.int32, device="cuda")
    q = torch.full((n * b, hkv * g, d), 5.0, device="cuda").half()
    big = torch.empty(64 << 20, dtype=torch.float32, device="cuda")
    for i in range(12):
        out = torch.full_like(q, 7.0)
        big.fill_(float(i))                       # the queries leave the caches
        o, lse = pa.paged_prompt_attention(q, k, k, table, starts, lens, 16, num_splits=1, out=out,
                                           return_lse=True)
        assert (o == 0).all() and (lse == -1e30).all(), f"pass {i}"


def test_prompt_of_one_token_is_decode():
    import paged_attention as pa
    lens, window, sinks = [1, 40, 700, 64], 100, 4
    c, q, st, o, lse = _run([1] * 4, lens, 8, 2, 128, 16, torch.bfloat16, window, sinks, seed=2)
    d, dl = pa.paged_attention(q, c.k, c.v, c.table, c.lens, 16, window=window, num_sinks=sinks,
                               return_lse=True)
    # probabilities rounded to 8 bits here and to 16 there
    assert_matches(o, d.double().cpu(), 2 * 2.0 ** -8 * c.v[~c.v.isnan()].abs().max().double().cpu()
                   * torch.ones(d.shape, dtype=torch.float64), "prompt against decode")
    assert_lse(lse, dl.double().cpu(), 128, "prompt against decode")


def test_prompt_strided_inputs():
    """K and V as slices of one buffer, a q that is a slice of a fused projection."""
    import paged_attention as pa
    qs, lens, bs, hkv, g, d, window, sinks = [50, 9], [200, 77], 16, 2, 4, 128, 60, 4
    c = PoisonedCache(lens, qs, hkv, d, bs, torch.float16, window, sinks, 3)
    kv = torch.stack([c.k, c.v], 1)
    fused = torch.randn(59, hkv * g + 2 * hkv, d, device="cuda").half()
    q = fused[:, : hkv * g]
    st = torch.tensor(_starts(qs), dtype=torch.int32, device="cuda")
    out = torch.empty(hkv * g, 59, d, device="cuda").half().transpose(0, 1)
    o = pa.paged_prompt_attention(q, kv[:, 0], kv[:, 1], c.table, st, c.lens, bs, window=window,
                                  num_sinks=sinks, out=out)
    want, _, tol = reference(q, c.k, c.v, c.table, lens, bs, window, sinks, _starts(qs))
    vmax = c.v[~c.v.isnan()].abs().max().double().item()
    assert o.data_ptr() == out.data_ptr()
    assert_matches(o, want, _tolerance(q, tol, vmax), "strided")


def test_prompt_large_scores_and_scale():
    """Scores in the hundreds, a running maximum that keeps growing, a given scale."""
    import paged_attention as pa
    qs, lens, bs, d = [64], [1024], 16, 128
    for dtype in (torch.float16, torch.bfloat16):
        c = PoisonedCache(lens, qs, 1, d, bs, dtype, 10 ** 9, 0, 5)
        ramp = torch.arange(1024, device="cuda") / 64.0
        page, slot = c.table[0, torch.arange(1024) // bs].long(), torch.arange(1024, device="cuda") % bs
        c.k[page, slot] = (c.k[page, slot].float() * ramp[:, None, None]).to(dtype)
        q = torch.randn(64, 4, d, device="cuda").to(dtype)
        st = torch.tensor([0, 64], dtype=torch.int32, device="cuda")
        o, lse = pa.paged_prompt_attention(q, c.k, c.v, c.table, st, c.lens, bs, scale=0.5,
                                           return_lse=True)
        want, wl, tol = reference(q, c.k, c.v, c.table, lens, bs, 10 ** 9, 0, [0, 64], scale=0.5)
        vmax = c.v[~c.v.isnan()].abs().max().double().item()
        assert_matches(o, want, _tolerance(q, tol, vmax), f"ramp {dtype}")


def test_prompt_captured_and_replayed_follows_lengths():
    import paged_attention as pa
    bs, hkv, g, d, window, sinks = 16, 2, 4, 128, 90, 4
    ws = pa.DecodeWorkspace("cuda")
    width, pool = 40, 128
    kk = torch.full((pool, bs, hkv, d), float("nan"), device="cuda").half()
    vv = kk.clone()
    table = torch.full((3, width), -1, dtype=torch.int32, device="cuda")
    st = torch.zeros(4, dtype=torch.int32, device="cuda")
    lens = torch.zeros(3, dtype=torch.int32, device="cuda")
    q = torch.randn(64, hkv * g, d, device="cuda").half()
    out = torch.zeros_like(q)

    def call():
        pa.paged_prompt_attention(q, kk, vv, table, st, lens, bs, window=window, num_sinks=sinks,
                                  workspace=ws, out=out)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for seed, (qs, ls) in enumerate([([20, 0, 44], [600, 3, 50]), ([1, 1, 1], [300, 640, 1]),
                                     ([64, 0, 0], [64, 0, 10])]):
        c = PoisonedCache(ls, qs, hkv, d, bs, torch.float16, window, sinks, seed, width=width)
        kk.fill_(float("nan"))
        vv.fill_(float("nan"))
        kk[: c.k.shape[0]], vv[: c.v.shape[0]] = c.k, c.v
        table.copy_(c.table)
        lens.copy_(c.lens)
        starts = _starts(qs)
        st.copy_(torch.tensor(starts, dtype=torch.int32))
        out.fill_(7)
        graph.replay()
        want, _, tol = reference(q, c.k, c.v, c.table, ls, bs, window, sinks, starts)
        vmax = c.v[~c.v.isnan()].abs().max().double().item()
        n = starts[-1]
        assert_matches(out[:n], want[:n], _tolerance(q, tol, vmax)[:n], f"replay {seed}")
        assert (out[n:] == 7).all()


def test_prompt_same_bits_on_every_run_and_stream():
    c, q, st, o, lse = _run([300, 20], [900, 40], 8, 2, 128, 16, torch.bfloat16, 500, 4, seed=8)
    import paged_attention as pa
    side = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            o2, lse2 = pa.paged_prompt_attention(q, c.k, c.v, c.table, st, c.lens, 16, window=500,
                                                 num_sinks=4, return_lse=True)
        side.synchronize()
        assert torch.equal(o, o2) and torch.equal(lse, lse2)


@pytest.mark.parametrize("count", [31, 32, 33, 300, 1200])
@pytest.mark.parametrize("d,bs", [(64, 16), (128, 8), (32, 16)])
def test_prompt_many_sequences(count, d, bs):
    """More sequences than a warp, than a block: empty ones, single tokens, small chunks."""
    qs = [(7 * i) % 5 if i % 11 else 23 for i in range(count)]
    lens = [q + (13 * i) % 70 for i, q in enumerate(qs)]
    _run(qs, lens, 4, 2, d, bs, torch.float16, 30, 3, seed=count + d, pad=5)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hkv,g,d,bs,q,s,window,sinks", [
    (2, 4, 128, 16, 1500, 3000, 1000, 4),
    (1, 8, 64, 32, 2000, 2001, None, 0),
    (4, 1, 128, 128, 900, 5000, 4097, 129),
    (2, 2, 256, 64, 700, 1400, 513, 65),
    (1, 5, 128, 8, 1025, 2050, 300, 1),
])
def test_prompt_long(dtype, hkv, g, d, bs, q, s, window, sinks):
    """Many key tiles, against products in 64 bits on the device."""
    import paged_attention as pa
    gen = torch.Generator(device="cuda").manual_seed(q)
    pages = -(-s // bs)
    k, v = (torch.randn(pages, bs, hkv, d, device="cuda", generator=gen).to(dtype) for _ in range(2))
    table = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)[None]
    x = torch.randn(q, hkv * g, d, device="cuda", generator=gen).to(dtype)
    lens = torch.tensor([s], dtype=torch.int32, device="cuda")
    st = torch.tensor([0, q], dtype=torch.int32, device="cuda")
    o, lse = pa.paged_prompt_attention(x, k, v, table, st, lens, bs, window=window,
                                       num_sinks=sinks, return_lse=True)
    t = torch.arange(s, device="cuda")
    pos = torch.arange(s - q, s, device="cuda")[:, None]
    seen = (t <= pos) & ((t < sinks) | (t > pos - (window or 10 ** 9)))
    kk, vv = (c[table[0].long()].reshape(-1, hkv, d)[:s].double() for c in (k, v))
    half, vmax = torch.finfo(dtype).eps / 2, vv.abs().max().item()
    for h in range(hkv * g):
        sc = (x[:, h].double() @ kk[:, h // g].T * d ** -0.5).masked_fill(~seen, float("-inf"))
        big = (x[:, h].double().abs() @ kk[:, h // g].abs().T * d ** -0.5).amax(1, keepdim=True)
        norm = torch.logsumexp(sc, 1, keepdim=True)
        want = (sc - norm).exp() @ vv[:, h // g]
        tol = half * want.abs() + (half + 2 * d * 2.0 ** -24 * big) * vmax
        assert_matches(o[:, h], want.cpu(), tol.cpu(), f"head {h}")
        assert_lse(lse[:, h], norm[:, 0].cpu(), d, f"head {h}")


def test_prompt_and_decode_on_two_streams_at_once():
    """Calls that share no workspace, running side by side, give what they give alone."""
    import paged_attention as pa
    jobs = []
    for i, (hkv, g, d) in enumerate([(2, 4, 128), (4, 2, 64), (2, 2, 256)]):
        qs, lens = [700, 3, 90], [900, 2000, 90]
        c = PoisonedCache(lens, qs, hkv, d, 16, torch.bfloat16, 400, 4, i)
        q = torch.randn(sum(qs), hkv * g, d, device="cuda").bfloat16()
        st = torch.tensor(_starts(qs), dtype=torch.int32, device="cuda")
        last = q[st[1:].long() - 1].contiguous()
        jobs.append((c, q, st, last))

    def both(job):
        c, q, st, last = job
        return (pa.paged_prompt_attention(q, c.k, c.v, c.table, st, c.lens, 16, window=400, num_sinks=4),
                pa.paged_attention(last, c.k, c.v, c.table, c.lens, 16, window=400, num_sinks=4))

    alone = [both(j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [[] for _ in jobs]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(both(jobs[i]))
    torch.cuda.synchronize()
    for want, outs in zip(alone, got):
        for o in outs:
            assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])


def test_prompt_flags_bad_pages_lengths_and_starts():
    import paged_attention as pa
    from paged_attention import _native
    for d, bs in ((64, 16), (32, 16)):
        c = PoisonedCache([200, 100], [10, 10], 1, d, bs, torch.float16, 50, 4, 3)
        q = torch.randn(20, 1, d, device="cuda").half()
        st = torch.tensor([0, 10, 20], dtype=torch.int32, device="cuda")
        ws = pa.DecodeWorkspace("cuda")

        def call(starts=st):
            pa.paged_prompt_attention(q, c.k, c.v, c.table, starts, c.lens, bs, window=50,
                                      num_sinks=4, workspace=ws)
            return ws.read_status()

        c.table[0, 5] = 10 ** 6                  # tokens 80..95: no row sees them
        assert call() == 0
        c.table[0, 11] = 10 ** 6                 # tokens 176..191: visible
        assert call() == _native.PA_STATUS_BAD_BLOCK
        c.table[0, 11] = -5
        ws.reset()
        assert call() == _native.PA_STATUS_BAD_BLOCK
        c.table[0, 11] = 0
        ws.reset()
        assert call(torch.tensor([0, 10, 21], dtype=torch.int32, device="cuda")) == \
            _native.PA_STATUS_BAD_SEQLEN
        ws.reset()
        assert call(torch.tensor([5, 3, 20], dtype=torch.int32, device="cuda")) & \
            _native.PA_STATUS_BAD_SEQLEN
        ws.reset()
        c.lens[1] = 10 ** 6
        assert call() & _native.PA_STATUS_BAD_SEQLEN


def test_prompt_empty_calls():
    import paged_attention as pa
    k = torch.zeros(4, 16, 2, 64, device="cuda", dtype=torch.float16)
    q = torch.zeros(0, 4, 64, device="cuda", dtype=torch.float16)
    bt = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    z = torch.zeros(3, dtype=torch.int32, device="cuda")
    o, lse = pa.paged_prompt_attention(q, k, k, bt, z, z[:2], 16, return_lse=True)
    assert o.shape == (0, 4, 64) and lse.shape == (0, 4)
    q = torch.zeros(5, 4, 64, device="cuda", dtype=torch.float16)
    out = torch.full_like(q, 3.0)
    pa.paged_prompt_attention(q, k, k, bt, z, z[:2], 16, out=out)          # rows of no sequence
    pa.paged_prompt_attention(q, k, k, bt[:0], z[:1], z[:0], 16, out=out)  # no sequence
    assert (out == 3).all()


def test_prompt_refusals_on_the_device():
    import paged_attention as pa
    k = torch.zeros(4, 16, 2, 64, device="cuda", dtype=torch.float16)
    q = torch.zeros(5, 4, 64, device="cuda", dtype=torch.float16)
    bt = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    st = torch.zeros(3, dtype=torch.int32, device="cuda")
    ok = dict(Q=q, K_Cache=k, V_Cache=k, Block_Table=bt, query_starts=st, seq_lens=st[:2], block_size=16)
    for bad in (dict(K_Cache=k.bfloat16()), dict(V_Cache=k[:3]), dict(Q=q[..., :32]), dict(Q=q[:, :3]),
                dict(Block_Table=bt.long()), dict(query_starts=st[:2]), dict(seq_lens=st),
                dict(seq_lens=st[:2].long()), dict(block_size=8), dict(K_Cache=k.cpu()),
                dict(Q=q.float(), K_Cache=k.float(), V_Cache=k.float()), dict(out=q[:4]),
                dict(window=0), dict(num_sinks=1), dict(num_splits=0), dict(scale=-1.0)):
        with pytest.raises(ValueError):
            pa.paged_prompt_attention(**{**ok, **bad})


def test_prompt_through_ctypes():
    from paged_attention import _native
    qs, lens, bs, hkv, d, window, sinks = [30, 4], [200, 900], 16, 2, 128, 70, 4
    c = PoisonedCache(lens, qs, hkv, d, bs, torch.bfloat16, window, sinks, 1)
    q = torch.randn(34, 4 * hkv, d, device="cuda").bfloat16()
    st = torch.tensor(_starts(qs), dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    p = _native.PromptParams()
    p.q, p.q_stride_t, p.q_stride_h = q.data_ptr(), q.stride(0), q.stride(1)
    p.k_cache, p.v_cache = c.k.data_ptr(), c.v.data_ptr()
    p.k_stride_block, p.k_stride_slot, p.k_stride_head = c.k.stride()[:3]
    p.v_stride_block, p.v_stride_slot, p.v_stride_head = c.v.stride()[:3]
    p.block_table, p.bt_stride_b, p.max_blocks = c.table.data_ptr(), c.table.stride(0), c.table.shape[1]
    p.query_starts, p.seq_lens = st.data_ptr(), c.lens.data_ptr()
    p.num_tokens, p.batch, p.num_heads, p.num_kv_heads, p.head_dim = 34, 2, 4 * hkv, hkv, d
    p.block_size, p.num_blocks, p.window, p.num_sinks = bs, c.k.shape[0], window, sinks
    p.scale, p.dtype = d ** -0.5, _native.PA_BF16
    p.out, p.out_stride_t, p.out_stride_h = out.data_ptr(), out.stride(0), out.stride(1)
    lib = _native.lib()
    need = ctypes.c_size_t()
    assert lib.pa_prompt_workspace(ctypes.byref(p), ctypes.byref(need)) == 0
    if need.value:
        assert lib.pa_prompt(ctypes.byref(p), None) == _native.PA_ERR_WORKSPACE
    buf = torch.empty(max(16, need.value), dtype=torch.uint8, device="cuda")
    p.workspace, p.workspace_bytes = buf.data_ptr(), need.value
    assert lib.pa_prompt(ctypes.byref(p), torch.cuda.current_stream().cuda_stream) == 0
    want, _, tol = reference(q, c.k, c.v, c.table, lens, bs, window, sinks, _starts(qs))
    vmax = c.v[~c.v.isnan()].abs().max().double().item()
    assert_matches(out, want, _tolerance(q, tol, vmax), "ctypes")


@pytest.mark.parametrize("splits", [1, 3, 40])
@pytest.mark.parametrize("d,bs,n,s", [(32, 16, 3, 700), (32, 16, 1, 1), (64, 16, 5, 700), (128, 16, 5, 700),
                                      (128, 16, 300, 700), (256, 32, 5, 700), (128, 5, 5, 700),
                                      (64, 16, 1, 1)])
def test_numbers_that_are_none_in_visible_places_show(d, bs, n, s, splits):
    """NaN or infinity in a visible key makes the rows that see it NaN, LSE included, in a
    visible value its dimension; the other KV head's rows keep their bits. The key's place
    runs through eight neighbours: a quarter of the exponentials is computed another way."""
    import paged_attention as pa
    g = torch.Generator().manual_seed(d + n)
    window, sinks = 350, 3
    pages = -(-s // bs)
    k, v = (torch.randn(pages, bs, 2, d, generator=g).half().cuda() for _ in range(2))
    q = torch.rand(n, 4, d, generator=g).half().cuda() + 0.01
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    starts = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    lens = torch.tensor([s], dtype=torch.int32, device="cuda")

    def run():
        return pa.paged_prompt_attention(q, k, v, table, starts, lens, bs, window=window, num_sinks=sinks,
                                         return_lse=True, num_splits=splits)
    clean, clean_lse = run()
    assert clean.isfinite().all()
    for t in [1] + [s - n - 20 + i for i in range(8)] if s > 1 else [0]:   # every row sees these
        for value in (float("nan"), float("inf")):
            kept = k[t // bs, t % bs, 0].clone()
            k[t // bs, t % bs, 0, 5] = value
            o, lse = run()
            k[t // bs, t % bs, 0] = kept
            assert o[:, :2].isnan().all() and lse[:, :2].isnan().all(), f"key {t} {value}"
            assert torch.equal(o[:, 2:], clean[:, 2:]) and torch.equal(lse[:, 2:], clean_lse[:, 2:])
        kept = v[t // bs, t % bs, 0].clone()
        v[t // bs, t % bs, 0, 7] = float("nan")
        o, lse = run()
        v[t // bs, t % bs, 0] = kept
        assert o[:, :2, 7].isnan().all(), f"value {t}"
        o[:, :2, 7] = clean[:, :2, 7]
        assert torch.equal(o, clean) and torch.equal(lse, clean_lse)


def _relayout(x, kind):
    """The same cache [NB, bs, Hkv, D] under other strides; what lies between is NaN."""
    nb, bs, hkv, d = x.shape
    nan = dict(fill_value=float("nan"), dtype=x.dtype, device=x.device)
    if kind == "heads first":
        y = torch.full((nb, hkv, bs, d), **nan).transpose(1, 2)
    elif kind == "half of pairs":
        y = torch.full((nb, 2, bs, hkv, d), **nan)[:, 1]
    elif kind == "head outermost":
        y = torch.full((hkv, nb, bs, d), **nan).permute(1, 2, 0, 3)
    elif kind == "padded rows":              # strides that are no whole numbers of rows
        y = torch.full((nb, bs, hkv, d + 8), **nan)[..., :d]
    elif kind == "padded pages":
        y = torch.full((nb, bs * hkv * d + 24), **nan)[:, : bs * hkv * d].unflatten(1, (bs, hkv, d))
    else:
        y = torch.full((nb, bs, hkv, d), **nan)
    y.copy_(x)
    return y


@pytest.mark.parametrize("bs", [1, 4, 12, 16])
@pytest.mark.parametrize("kinds", [("plain", "heads first"), ("half of pairs", "head outermost"),
                                   ("padded rows", "padded rows"), ("plain", "padded pages")])
@pytest.mark.parametrize("hkv,d", [(2, 128), (1, 64), (3, 256), (3, 32)])
def test_prompt_cache_layouts(bs, kinds, hkv, d):
    """Every way the keys' rows are fetched gives the bits of the plain layout."""
    import paged_attention as pa
    qs, lens, window, sinks = [170, 1, 33], [400, 77, 33], 90, 5
    c = PoisonedCache(lens, qs, hkv, d, bs, torch.float16, window, sinks, bs + d)
    q = torch.randn(204, hkv * 3, d, device="cuda").half()
    st = torch.tensor(_starts(qs), dtype=torch.int32, device="cuda")
    outs = [pa.paged_prompt_attention(q, k, v, c.table, st, c.lens, bs, window=window, num_sinks=sinks)
            for k, v in ((c.k, c.v), (_relayout(c.k, kinds[0]), _relayout(c.v, kinds[1])))]
    want, _, tol = reference(q, c.k, c.v, c.table, lens, bs, window, sinks, _starts(qs))
    vmax = c.v[~c.v.isnan()].abs().max().double().item()
    assert_matches(outs[0], want, _tolerance(q, tol, vmax), "plain")
    assert torch.equal(outs[0], outs[1])


def test_prompt_pool_of_one_token():
    import paged_attention as pa
    for d in (64, 128, 256):
        k, v = (torch.randn(1, 1, 1, d, device="cuda").half() for _ in range(2))
        st = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
        o = pa.paged_prompt_attention(torch.randn(1, 2, d, device="cuda").half(), k, v,
                                      torch.zeros(1, 1, dtype=torch.int32, device="cuda"), st,
                                      st[1:], 1)
        assert torch.equal(o, v[0, 0].expand(1, 2, d))


@pytest.mark.parametrize("splits", [1, 2, 5])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [32, 64, 128, 256])
def test_prompt_lse_of_large_scores(d, dtype, splits):
    """Scores in the hundreds under a maximum that keeps growing: the LSE, whose sum is kept
    against an older maximum, alone and joined from parts with LSEs far apart.

    Tolerance: each score's rounding in 32 bits, 2^-24 D sum|q_i k_i| scale; the scaled maximum,
    its difference to a score and the parts' LSEs, each rounded a few times (8 * 2^-24 of the
    largest score or LSE); exponentials and the sum of 1024, 1e-5 relative at most."""
    import paged_attention as pa
    n, s, bs = 64, 1024, 16
    c = PoisonedCache([s], [n], 1, d, bs, dtype, 10 ** 9, 0, 5)
    ramp = torch.arange(s, device="cuda") / 64.0
    page, slot = c.table[0, torch.arange(s) // bs].long(), torch.arange(s, device="cuda") % bs
    c.k[page, slot] = (c.k[page, slot].float() * ramp[:, None, None]).to(dtype)
    q = torch.randn(n, 4, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(d)).to(dtype)
    st = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    o, lse = pa.paged_prompt_attention(q, c.k, c.v, c.table, st, c.lens, bs, scale=0.5, return_lse=True,
                                       num_splits=splits)
    want, wl, tol = reference(q, c.k, c.v, c.table, [s], bs, 10 ** 9, 0, [0, n], scale=0.5)
    vmax = c.v[~c.v.isnan()].abs().max().double().item()
    assert_matches(o, want, _tolerance(q, tol, vmax), "O")
    big = (q.double().abs().cpu() @ c.k[page, slot, 0].double().abs().cpu().T * 0.5).amax(-1)
    bound = d * 2.0 ** -24 * big + 8 * 2.0 ** -24 * torch.maximum(wl.abs(), big) + 1e-5
    assert not ((lse.double().cpu() - wl).abs() > bound).any(), (lse.double().cpu() - wl).abs().max()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("g", [1, 4])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("fma_columns", [True, False])
def test_prompt_exponentials(d, g, dtype, fma_columns):
    """The sum of exponentials by itself: queries of a single one and keys of the scores wanted,
    so that the scores are exact. They sit in the columns (of each eight, two) whose exponentials
    are a polynomial on the FMA pipe, or in the others; token 0 holds the maximum, 0.

    Tolerance of the LSE = log(1 + sum of the others), all relative errors of a sum of positive
    terms: the polynomial's 2.9e-6 or ex2's 2^-22; the argument, rounded from |x| up to 20,
    3 * 2^-24 |x| e^x <= 3 * 2^-24; 32 additions a lane, 3 across them and one per tile of 512
    tokens at most; the result's own 4 * 2^-24 (1 + |LSE|)."""
    import paged_attention as pa
    s, bs = 512, 16
    n = s + d
    gen = torch.Generator().manual_seed(d + g)
    x = torch.full((n, d), -100.0)
    cols = torch.tensor([t for t in range(1, s) if ((t & 6) == 4) == fma_columns])
    x[cols] = -20 * torch.rand(len(cols), d, generator=gen) ** 2
    x[0] = 0
    x = x.to(dtype)
    k = x.view(n // bs, bs, 1, d).cuda()
    q = torch.eye(d).to(dtype).cuda()[:, None].expand(d, g, d)
    table = torch.arange(n // bs, dtype=torch.int32, device="cuda")[None]
    st = torch.tensor([0, d], dtype=torch.int32, device="cuda")
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    _, lse = pa.paged_prompt_attention(q, k, k, table, st, lens, bs, scale=1.0, return_lse=True, num_splits=1)
    want = torch.logsumexp(x.double()[: s + 1], 0)[:, None]      # (the rest weighs e^-100)
    ulp = 2.0 ** -24
    tol = (2.9e-6 if fma_columns else 2.0 ** -22) + 3 * ulp + (32 + 3 + 9) * ulp + 4 * ulp * (1 + want.abs())
    err = (lse.double().cpu() - want).abs()
    assert not (err > tol).any(), f"off by {err.max().item():.2e}, allowed {tol.min().item():.2e}"


def test_prompt_captured_graph_outlives_a_growing_workspace():
    """A call that grows the workspace leaves a graph captured before it with its own scratch;
    what is allocated in between is not written by the replay."""
    import paged_attention as pa
    qs, lens, window, sinks = [5, 3], [900, 700], 600, 4
    c = PoisonedCache(lens, qs, 2, 128, 16, torch.float16, window, sinks, 3)
    q = torch.randn(8, 8, 128, device="cuda").half()
    st = torch.tensor(_starts(qs), dtype=torch.int32, device="cuda")
    ws = pa.DecodeWorkspace("cuda")
    out = torch.zeros_like(q)

    def call(splits):
        pa.paged_prompt_attention(q, c.k, c.v, c.table, st, c.lens, 16, window=window, num_sinks=sinks,
                                  workspace=ws, out=out, num_splits=splits)
    call(3)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(3)
    graph.replay()
    want = out.clone()
    size = ws.buffer.numel()
    call(40)
    assert ws.buffer.numel() > size
    others = [torch.full((size,), 7, dtype=torch.uint8, device="cuda") for _ in range(8)]
    out.zero_()
    graph.replay()
    assert torch.equal(out, want)
    assert all((x == 7).all() for x in others)
