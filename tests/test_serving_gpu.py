"""The windowed operators used together, as a serving loop does: pages taken and given
back by ``PagePool``, K and V written by ``write_kv_cache``, prompts in chunks by
``paged_prompt_attention``, single tokens by ``paged_attention``, continuations by
``fork``, the pool moved together by ``compact``. Each step's output is compared with
attention over the whole history of each stream, kept apart on the CPU."""
import pytest
import torch

from window_helpers import assert_matches, reference

pytestmark = pytest.mark.gpu


class Streams:
    def __init__(self, rows, pool_pages, bs, layers, hkv, g, d, dtype, window, sinks, seed):
        import paged_attention as pa
        self.pa = pa
        self.gen = torch.Generator().manual_seed(seed)
        self.bs, self.layers, self.hkv, self.g, self.d = bs, layers, hkv, g, d
        self.dtype, self.window, self.sinks = dtype, window, sinks
        nan = float("nan")
        self.k = [torch.full((pool_pages, bs, hkv, d), nan, device="cuda").to(dtype) for _ in range(layers)]
        self.v = [torch.full((pool_pages, bs, hkv, d), nan, device="cuda").to(dtype) for _ in range(layers)]
        self.pool = pa.PagePool(self.k, self.v)
        self.table = torch.full((rows, 64), -1, dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(rows, dtype=torch.int32, device="cuda")
        self.history = [[[] for _ in range(layers)] for _ in range(rows)]     # (k, v) per token

    def _rand(self, *shape):
        return torch.randn(*shape, generator=self.gen).to(self.dtype)

    def step(self, new):
        """`new[r]` new tokens of row r; attention from each of them, in every layer."""
        before = self.lens.tolist()
        target = [s + n if n else -1 for s, n in zip(before, new)]
        self.pool.resize(self.table, self.lens,
                         torch.tensor(target, dtype=torch.int32, device="cuda"),
                         window=self.window, num_sinks=self.sinks)
        rows = [r for r, n in enumerate(new) if n]
        starts = [0]
        for r in rows:
            starts.append(starts[-1] + new[r])
        pos = torch.tensor([before[r] + i for r in rows for i in range(new[r])], device="cuda")
        owner = torch.tensor([r for r in rows for _ in range(new[r])], device="cuda")
        slots = self.table[owner, pos // self.bs].long() * self.bs + pos % self.bs
        at = torch.tensor(rows, device="cuda")
        sub, lens = self.table[at], self.lens[at]
        one = all(new[r] == 1 for r in rows)
        for layer in range(self.layers):
            k, v = self._rand(len(pos), self.hkv, self.d), self._rand(len(pos), self.hkv, self.d)
            q = self._rand(len(pos), self.hkv * self.g, self.d)
            i = 0
            for r in rows:
                for _ in range(new[r]):
                    self.history[r][layer].append((k[i], v[i]))
                    i += 1
            self.pa.write_kv_cache(k.cuda(), v.cuda(), self.k[layer], self.v[layer], slots)
            if one:
                o = self.pa.paged_attention(q.cuda(), self.k[layer], self.v[layer], sub, lens, self.bs,
                                            window=self.window, num_sinks=self.sinks)
            else:
                o = self.pa.paged_prompt_attention(
                    q.cuda(), self.k[layer], self.v[layer], sub,
                    torch.tensor(starts, dtype=torch.int32, device="cuda"), lens, self.bs,
                    window=self.window, num_sinks=self.sinks)
            self._check(o, q, rows, starts, layer)
        assert self.pool.read_status() == 0

    def _check(self, o, q, rows, starts, layer):
        """Against the histories, as one page per row."""
        longest = max(len(self.history[r][layer]) for r in rows)
        k = torch.zeros(len(rows), longest, self.hkv, self.d, dtype=self.dtype)
        v = torch.zeros_like(k)
        lens = []
        for i, r in enumerate(rows):
            h = self.history[r][layer]
            k[i, : len(h)] = torch.stack([x for x, _ in h])
            v[i, : len(h)] = torch.stack([x for _, x in h])
            lens.append(len(h))
        table = torch.arange(len(rows))[:, None]
        want, _, tol = reference(q, k, v, table, lens, longest, self.window, self.sinks, starts)
        # probabilities rounded to half a step in the prompt form
        tol = tol + torch.finfo(self.dtype).eps / 2 * v.abs().max().double()
        assert_matches(o, want, tol, f"rows {rows} layer {layer}")

    def end(self, r):
        new = [-1] * len(self.history)
        new[r] = 0
        self.pool.resize(self.table, self.lens, torch.tensor(new, dtype=torch.int32, device="cuda"))
        self.history[r] = [[] for _ in range(self.layers)]

    def fork(self, parents, children):
        t = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (parents, children)]
        self.pool.fork(self.table, self.lens, *t)
        for p, c in zip(parents, children):
            self.history[c] = [list(h) for h in self.history[p]]

    def cut(self, r, tokens):
        """Rejected draft tokens are taken back."""
        new = [-1] * len(self.history)
        new[r] = int(self.lens[r]) - tokens
        self.pool.resize(self.table, self.lens, torch.tensor(new, dtype=torch.int32, device="cuda"),
                         window=self.window, num_sinks=self.sinks)
        for h in self.history[r]:
            del h[-tokens:]


@pytest.mark.parametrize("dtype,bs,hkv,g,d,window,sinks", [
    (torch.bfloat16, 16, 2, 4, 128, 40, 4),
    (torch.float16, 8, 1, 2, 64, 24, 3),
    (torch.float16, 32, 2, 1, 128, 70, 0),
])
def test_streams_beyond_their_window(dtype, bs, hkv, g, d, window, sinks):
    s = Streams(6, 60, bs, 2, hkv, g, d, dtype, window, sinks, seed=bs)
    s.step([70, 5, 130, 0, 0, 0])                  # prompts
    s.step([33, 0, 64, 0, 0, 0])                   # their second chunks
    for _ in range(3):
        s.step([1, 1, 1, 0, 0, 0])
    s.fork([0, 0, 1], [3, 4, 5])                   # continuations
    for _ in range(bs + 2):
        s.step([1, 1, 1, 1, 1, 1])
    s.end(0)
    s.end(2)
    live = int(s.pool.compact(s.table))
    assert live == int((s.pool.refs > 0).sum())
    assert not s.pool.refs[live:].any()
    for _ in range(2):
        s.step([0, 1, 0, 1, 1, 1])
    s.step([25, 0, 3, 4, 1, 2])                    # a new prompt beside drafts
    s.cut(3, 2)
    s.step([1, 1, 1, 1, 1, 1])
    for r in range(6):
        s.end(r)
    torch.cuda.synchronize()
    assert int(s.pool.refs.abs().sum()) == 0 and s.pool.read_status() == 0
