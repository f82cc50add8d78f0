"""The operators of a batched step together, as a serving loop uses them: prompts, then sampled tokens, with sequences that
end, wait and return; captured into a graph; on streams of their own; and far into large buffers.  Each stage against its
64-bit form on what the stage before it gave, or bit for bit against the same work done another way."""
import numpy as np
import pytest

import fence_ops as F
import serving_ref as R
from gpu_util import LIVE, dev, host, stream, torch_mod
from test_gpu_serving import HEADS, bound, check_attention, empty, pages_of, run_attention

pytestmark = pytest.mark.gpu


class Loop:
    """A serving loop of one attention layer without weights: a token's q, k and v are its row of a table, and the
    attention's output is its logits."""
    HEADS, KVH, D, PAGE, BLOCKS = 8, 2, 64, 16, 12

    def __init__(self, batch, pages, rows, cache, half, seed):
        torch = torch_mod()
        rng = np.random.default_rng(seed)
        self.batch, self.pages, self.rows, self.cache, self.half = batch, pages, rows, cache, half
        self.vocab = self.HEADS * self.D
        i32 = lambda *s: empty(s, torch.int32, 0)  # noqa: E731
        self.table = dev(rng.standard_normal((self.vocab, self.HEADS + 2 * self.KVH, self.D)).astype(np.float32))
        self.norm = dev(rng.standard_normal((2, self.D)).astype(np.float32) * 0.1 + 1)
        self.codes = empty((2, pages, self.KVH, self.PAGE, self.D), torch.uint8, 0)
        self.scale = empty((2, pages, self.KVH), torch.float32, 0)
        self.lens, self.new, self.admitted, self.tok = i32(batch), i32(batch), i32(batch), i32(batch)
        self.blocks, self.q_start = i32(batch, self.BLOCKS), i32(batch + 1)
        self.free, self.count = dev(rng.permutation(pages).astype(np.int32)), dev(np.array([pages], np.int32))
        self.positions, self.slots, self.tokens = i32(rows), i32(rows), i32(rows)
        self.out = empty((rows, self.vocab), torch.float16 if half else torch.float32, 0)
        self.temperature = dev(np.resize(np.array([0.7, 0, 1.3, 0.05], np.float32), batch))
        self.top_k = dev(np.resize(np.array([0, 5, 40], np.int32), batch))
        self.top_p = dev(np.resize(np.array([0.9, 1.0], np.float32), batch))
        self.u, self.drawn = empty((batch,), torch.float32, 0), i32(batch)
        self.at_size = F.gqa_attention_q8_workspace(batch, rows, self.HEADS, self.KVH, self.D)
        self.ws_size = F.sample_workspace(batch, self.vocab)
        self.at_ws, self.ws = empty((self.at_size,), torch.uint8, 255), empty((self.ws_size,), torch.uint8, 255)

    def plan(self):
        p = lambda t: t.data_ptr()  # noqa: E731
        F.kv_plan(p(self.lens), p(self.lens), p(self.new), self.batch, p(self.blocks), self.BLOCKS, self.PAGE, p(self.free),
                  p(self.count), p(self.count), self.pages, p(self.q_start), p(self.positions), p(self.slots), self.rows,
                  p(self.admitted), stream())

    def step(self, max_q):
        """Everything behind the plan, of self.tokens."""
        torch = torch_mod()
        x = self.table[self.tokens.long()]
        h, kv = self.HEADS, self.KVH
        self.q, self.k = x[:, :h].contiguous(), x[:, h:h + kv].contiguous()
        self.v = x  # the v heads stay in the fused row
        F.qk_norm_rope(self.q.data_ptr(), self.k.data_ptr(), self.norm[0].data_ptr(), self.norm[1].data_ptr(), self.rows, h, kv,
                       self.D, 1e-6, self.positions.data_ptr(), 0, 1e4, F.ROPE_NEOX, stream())
        self.kv = torch.cat([self.k, x[:, h + kv:]], 1)  # k and v as parts of one row
        pages = pages_of(self.codes, self.scale, self.cache)
        F.store_kv_q8(pages, self.kv.data_ptr(), self.kv[:, kv:].data_ptr(), F.F32, 2 * kv * self.D, self.slots.data_ptr(),
                      self.rows, stream())
        q = self.q.half() if self.half else self.q
        self.q_in = q
        F.gqa_attention_q8(self.out.data_ptr(), q.data_ptr(), F.F16 if self.half else F.F32, self.vocab, self.vocab, pages,
                           self.blocks.data_ptr(), self.BLOCKS, self.lens.data_ptr(), self.q_start.data_ptr(), self.batch,
                           max_q, h, self.at_ws.data_ptr(), self.at_size, stream())
        last = (self.q_start[1:] - 1).clamp(min=0).long()
        self.logits = self.out[last].float() * 8
        F.sample(self.drawn.data_ptr(), self.logits.data_ptr(), self.batch, self.vocab, self.vocab, self.temperature.data_ptr(),
                 self.top_k.data_ptr(), self.top_p.data_ptr(), 0, self.u.data_ptr(), self.ws.data_ptr(), self.ws_size, stream())
        self.tok.copy_(torch.where((self.new > 0) & (self.admitted > 0), self.drawn, self.tok))

    def place_tokens(self):
        """One token a sequence, the one drawn last, to its row."""
        torch = torch_mod()
        seq = torch.searchsorted(self.q_start[1:], self.arange, right=True).clamp(max=self.batch - 1)
        self.tokens.copy_(self.tok[seq])

    def state(self):
        return [host(t) for t in (self.lens, self.blocks, self.free, self.count, self.q_start, self.positions, self.slots,
                                  self.admitted, self.codes, self.scale, self.tok, self.drawn)]


@pytest.mark.parametrize("cache,half", [(R.INT8, False), (R.E4M3, True), (R.INT8, True)])
def test_serving_loop(cache, half):
    rng = np.random.default_rng(3 + half + cache)
    batch, rows = 6, 96
    loop = Loop(batch, 14, rows, cache, half, 5)
    # tokens of each sequence in each step; -1 ends it
    steps = [[20, 0, 33, 1, 0, 7], [1, 40, 1, 1, 0, 3], [1, 1, -1, 1, 50, 1], [1, 1, 17, 5, 1, -1], [0, 1, 1, 1, 1, 60],
             [1, 1, 1, 1, 1, 1], [-1, -1, 1, 90, 1, 1], [1, 5, 1, 1, 1, 1]]
    lens, table = np.zeros(batch, np.int32), np.zeros((batch, loop.BLOCKS), np.int32)
    free, count = host(loop.free).copy(), loop.pages
    refused = 0
    for new in steps:
        before = {"codes": host(loop.codes).copy(), "scale": host(loop.scale).copy(), "out": host(loop.out).copy()}
        tok = host(loop.tok).copy()
        tokens = np.zeros(rows, np.int32)
        at = 0
        for b, n in enumerate(new):
            tokens[at:at + max(n, 0)] = tok[b] if n == 1 else rng.integers(0, loop.vocab, max(n, 0))
            at += max(n, 0)
        u = rng.random(batch).astype(np.float32)
        torch = torch_mod()
        loop.new.copy_(torch.tensor(new, dtype=torch.int32))
        loop.tokens.copy_(torch.from_numpy(tokens))
        loop.u.copy_(torch.from_numpy(u))
        loop.plan()
        loop.step(rows)
        want = R.plan(lens, new, table, loop.PAGE, free, count, rows)  # changes table and free
        lens, count = np.asarray(want["lens"], np.int32), int(want["count"])
        for name, t in (("lens", loop.lens), ("q_start", loop.q_start), ("positions", loop.positions), ("slots", loop.slots),
                        ("admitted", loop.admitted)):
            assert np.array_equal(host(t), np.asarray(want[name])), name
        assert host(loop.count)[0] == count
        assert np.array_equal(host(loop.blocks), table) and np.array_equal(host(loop.free), free)
        refused += int((np.asarray(want["admitted"]) == 0).sum())
        kv = host(loop.kv).reshape(rows, 2, loop.KVH, loop.D)
        codes, scale = before["codes"], before["scale"]
        for i in range(2):
            R.store(codes[i], scale[i], kv[:, i], want["slots"], cache)
            assert np.array_equal(host(loop.codes)[i], codes[i]) and np.array_equal(host(loop.scale)[i], scale[i])
        got = host(loop.out).reshape(rows, loop.HEADS, loop.D)
        q = host(loop.q_in)
        exact, spread, big = R.attention(q, codes, scale, table, lens, want["q_start"], cache, rows)
        used = int(want["q_start"][-1])
        seen = np.repeat(np.asarray(want["admitted"]) > 0, np.diff(want["q_start"]))
        off = np.abs(got[:used].astype(np.float64) - exact[:used])
        most = bound(exact[:used], spread[:used], big[:used], loop.D, int(lens.max()), half, R.TOP[cache] * scale[1].max())
        assert (off <= most)[seen].all()
        assert np.array_equal(got[used:], before["out"].reshape(got.shape)[used:])  # the padding
        x = host(loop.logits)
        drawn = [R.sample(x[b], host(loop.temperature)[b], host(loop.top_k)[b], host(loop.top_p)[b], 0.0, u[b])
                 for b in range(batch)]
        assert host(loop.drawn).tolist() == drawn
    assert refused >= 1


def test_captured_step_replayed():
    """A step of single tokens at a fixed number of rows, captured once and replayed while sequences end, wait and return,
    with the program's own work and synchronisations between, equals the same steps run directly, bit for bit."""
    torch = torch_mod()
    rng = np.random.default_rng(8)
    batch, rows = 12, 16  # more rows than sequences: padding
    a, b = (Loop(batch, 60, rows, R.E4M3, True, 9) for _ in range(2))
    for s in (a, b):
        s.arange = torch.arange(rows, dtype=torch.int32, device="cuda")
        LIVE.append(s.arange)
        s.new.fill_(1)

    def one(s):
        s.plan()
        s.place_tokens()
        s.step(1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # a step of each before the capture, the same for both
        one(a)
        one(b)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one(a)
    for x, y in zip(a.state(), b.state()):
        assert np.array_equal(x, y)
    for step in range(30):
        new = torch.from_numpy(rng.choice([1, 1, 1, 1, 0, -1], batch).astype(np.int32))
        u = torch.from_numpy(rng.random(batch).astype(np.float32))
        for s in (a, b):
            s.new.copy_(new)
            s.u.copy_(u)
        if step % 3:
            torch.cuda.synchronize()
        graph.replay()
        one(b)
        if step % 5 == 0:
            LIVE.append(torch.full((1000, step + 1), 7.0, device="cuda"))
        for x, y in zip(a.state(), b.state()):
            assert np.array_equal(x, y), step
        used = int(host(a.q_start)[-1])
        assert torch.equal(a.out[:used], b.out[:used])


def test_calls_on_two_streams():
    """Calls that overlap on two streams, each with its own workspace, equal the same calls one after another."""
    torch = torch_mod()
    rng = np.random.default_rng(4)
    heads, kvh, d, page, cache = 16, 4, 128, 64, R.INT8
    jobs = []
    for kv_lens, q_lens, rows, vocab in (([20000, 17, 900], [1, 1, 4], 3, 50001), ([5000, 3000], [200, 1], 40, 20000)):
        blocks = max(-(-n // page) for n in kv_lens)
        table = np.arange(len(kv_lens) * blocks, dtype=np.int32).reshape(len(kv_lens), blocks)
        codes = rng.integers(-127, 128, (2, table.size, kvh, page, d)).astype(np.int8).view(np.uint8)
        scale = (rng.random((2, table.size, kvh)) * 0.02).astype(np.float32)
        q_start = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
        size = F.gqa_attention_q8_workspace(len(kv_lens), max(q_lens), heads, kvh, d)
        ssize = F.sample_workspace(rows, vocab)
        jobs.append(dict(
            n=len(kv_lens), most=max(q_lens), blocks=blocks, rows=rows, vocab=vocab, size=size, ssize=ssize, table=dev(table),
            codes=dev(codes), scale=dev(scale), q_start=dev(q_start), kv=dev(np.array(kv_lens, np.int32)),
            q=dev(rng.standard_normal((int(q_start[-1]), heads, d)).astype(np.float32)),
            x=dev((rng.standard_normal((rows, vocab)) * 3).astype(np.float32)), u=dev(rng.random(rows).astype(np.float32)),
            p=dev(np.full(rows, 0.95, np.float32)), t=dev(np.full(rows, 0.8, np.float32)),
            ws=empty((size,), torch.uint8, 255), sws=empty((ssize,), torch.uint8, 255)))

    def call(j, out, drawn):
        F.gqa_attention_q8(out.data_ptr(), j["q"].data_ptr(), F.F32, heads * d, heads * d, pages_of(j["codes"], j["scale"], cache),
                           j["table"].data_ptr(), j["blocks"], j["kv"].data_ptr(), j["q_start"].data_ptr(), j["n"], j["most"],
                           heads, j["ws"].data_ptr(), j["size"], stream())
        F.sample(drawn.data_ptr(), j["x"].data_ptr(), j["rows"], j["vocab"], j["vocab"], j["t"].data_ptr(), 0, j["p"].data_ptr(),
                 0, j["u"].data_ptr(), j["sws"].data_ptr(), j["ssize"], stream())

    outs = lambda j: (torch.full_like(j["q"], 7.0), torch.full((j["rows"],), -9, dtype=torch.int32, device="cuda"))  # noqa: E731
    want = [outs(j) for j in jobs]
    got = [[outs(j) for j in jobs] for _ in range(6)]
    LIVE.append((want, got))
    for j, o in zip(jobs, want):
        call(j, *o)
        torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for turn in got:
        for j, o, s in zip(jobs, turn, streams):
            with torch.cuda.stream(s):
                call(j, *o)
    torch.cuda.synchronize()
    for turn in got:
        for (x, y), (wx, wy) in zip(turn, want):
            assert torch.equal(x, wx) and torch.equal(y, wy)


@pytest.mark.parametrize("cache,half", [(R.INT8, False), (R.E4M3, True)])
def test_pages_past_32_bits(cache, half):
    """The same rows through pages at the two ends of a pool whose codes pass 4 GiB, and through a small pool."""
    torch = torch_mod()
    rng = np.random.default_rng(12)
    heads, kvh, d, page, n_pages = 16, 8, 128, 256, 17000  # 4.15 GiB of K codes and as many of V
    kv_lens, q_lens = [700, 300], [1, 40]
    ids = np.array([[0, n_pages - 1, 8191], [n_pages - 2, 8192, 0]], np.int32)
    small = np.array([[0, 4, 1], [3, 2, 0]], np.int32)
    dtype = np.float16 if half else np.float32
    k, v = ((rng.standard_normal((1000, kvh, d)) * 2).astype(dtype) for _ in range(2))
    q = rng.standard_normal((41, heads, d)).astype(dtype)
    d_k, d_v, d_q = dev(k), dev(v), dev(q)
    results = []
    for table, pages in ((ids, n_pages), (small, 5)):
        if pages == 5:
            codes, scale = empty((2, pages, kvh, page, d), torch.uint8, 0), empty((2, pages, kvh), torch.float32, 0)
        else:
            codes = torch.empty((2, pages, kvh, page, d), dtype=torch.uint8, device="cuda")
            scale = torch.zeros((2, pages, kvh), device="cuda")
            LIVE.append((codes, scale))
        slots = np.concatenate([table[b, np.arange(n) // page] * page + np.arange(n) % page for b, n in enumerate(kv_lens)])
        cp = pages_of(codes, scale, cache)
        F.store_kv_q8(cp, d_k.data_ptr(), d_v.data_ptr(), F.F16 if half else F.F32, kvh * d, dev(slots.astype(np.int32)).data_ptr(),
                      1000, stream())
        out = empty((41, heads, d), torch.float16 if half else torch.float32, 0)
        size = F.gqa_attention_q8_workspace(2, 40, heads, kvh, d)
        ws = empty((size,), torch.uint8, 255)
        F.gqa_attention_q8(out.data_ptr(), d_q.data_ptr(), F.F16 if half else F.F32, heads * d, heads * d, cp, dev(table).data_ptr(),
                           3, dev(np.array(kv_lens, np.int32)).data_ptr(), dev(np.array([0, 1, 41], np.int32)).data_ptr(), 2, 40,
                           heads, ws.data_ptr(), size, stream())
        at = torch.from_numpy(np.concatenate([table[0], table[1, :2]]).astype(np.int64)).cuda()
        used = codes[:, at]
        used[:, 2, :, 700 - 512:], used[:, 4, :, 300 - 256:] = 0, 0  # behind the last rows: whatever was there
        results.append((host(used).copy(), host(scale[:, at]).copy(), host(out).copy()))
    for x, y in zip(*results):
        assert np.array_equal(x, y)
    assert np.abs(results[0][2].astype(np.float64)).max() > 0.01


def test_rows_far_apart():
    """Rows of logits, q, k, v and out whose distance takes them past 32 bits of bytes and of elements."""
    torch = torch_mod()
    rng = np.random.default_rng(1)
    ld = 2 ** 30 + 2 ** 20  # two rows on: past 2^31 elements
    heads, kvh, d, page = 4, 2, 64, 16
    far = torch.empty(2 * ld + 4096, device="cuda")
    out = torch.empty(2 * ld + 4096, dtype=torch.float16, device="cuda")
    LIVE.append((far, out))
    x = (rng.standard_normal((3, 4096)) * 3).astype(np.float32)
    for r in range(3):
        far[r * ld:r * ld + 4096] = torch.from_numpy(x[r]).cuda()
    size = F.sample_workspace(3, 4096)
    ws, drawn = empty((size,), torch.uint8, 255), empty((3,), torch.int32, -9)
    u = np.array([0.3, 0.6, 0.9], np.float32)
    F.sample(drawn.data_ptr(), far.data_ptr(), 3, 4096, ld, 0, 0, 0, 0, dev(u).data_ptr(), ws.data_ptr(), size, stream())
    assert host(drawn).tolist() == [R.sample(x[r], u=u[r]) for r in range(3)]
    # the rows' first values as k and v (fp32), then as q and out (binary16)
    codes, scale = empty((2, 1, kvh, page, d), torch.uint8, 0), empty((2, 1, kvh), torch.float32, 0)
    pages = pages_of(codes, scale, R.INT8)
    F.store_kv_q8(pages, far.data_ptr(), far.data_ptr() + 4 * kvh * d, F.F32, ld, dev(np.arange(3, dtype=np.int32)).data_ptr(), 3,
                  stream())
    want, want_scale = np.zeros((2, 1, kvh, page, d), np.uint8), np.zeros((2, 1, kvh), np.float32)
    for i in range(2):
        R.store(want[i], want_scale[i], x[:, i * kvh * d:(i + 1) * kvh * d].reshape(3, kvh, d), np.arange(3), R.INT8)
    assert np.array_equal(host(codes), want) and np.array_equal(host(scale), want_scale)
    for r in range(3):
        out[r * ld:r * ld + heads * d] = torch.from_numpy(x[r, :heads * d]).cuda().half()
    q = np.stack([host(out[r * ld:r * ld + heads * d]) for r in range(3)]).reshape(3, heads, d)
    wsz = F.gqa_attention_q8_workspace(1, 3, heads, kvh, d)
    aws = empty((wsz,), torch.uint8, 255)
    table = np.zeros((1, 1), np.int32)
    F.gqa_attention_q8(out.data_ptr() + 2 * heads * d, out.data_ptr(), F.F16, ld, ld, pages, dev(table).data_ptr(), 1,
                       dev(np.array([3], np.int32)).data_ptr(), dev(np.array([0, 3], np.int32)).data_ptr(), 1, 3, heads,
                       aws.data_ptr(), wsz, stream())
    got = np.stack([host(out[r * ld + heads * d:r * ld + 2 * heads * d]) for r in range(3)]).reshape(3, heads, d)
    near = run_attention(q, want, want_scale, table, [3], [0, 3], R.INT8, True, 3)
    assert np.array_equal(got.astype(np.float64), near)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("cache", [R.INT8, R.E4M3])
def test_attention_large_batches(half, cache):
    """More sequences than the walk's chunk of the batch, most of them short, with idle and empty ones between."""
    rng = np.random.default_rng(31 + half + 2 * cache)
    for batch in (65, 257, 1030):
        kv = rng.integers(0, 40, batch)
        q = np.minimum(rng.choice([0, 1, 1, 1, 3], batch), kv)
        kv[batch // 2], q[batch // 2] = 900, 70
        check_attention(rng, 4, 2, 32, 16, kv, q, cache, half)


@pytest.mark.parametrize("pad", [1, 2, 3, 5])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("heads,kvh,d", [(8, 2, 64), (5, 1, 80)])
def test_attention_rows_at_odd_distances(heads, kvh, d, half, pad):
    """ldq and ldo that leave rows at their type's alignment and no more."""
    rng = np.random.default_rng(pad * 10 + d + half)
    check_attention(rng, heads, kvh, d, 32, [100, 33, 260], [1, 5, 90], R.INT8, half, pad=pad)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("heads,kvh,d", HEADS)
def test_attention_drafts(heads, kvh, d, half):
    """As many drafted tokens as one tile of columns holds, and one more."""
    rng = np.random.default_rng(heads + 3 * d + half)
    most = 16 * kvh // heads
    for q in ([most, 1, most], [most + 1, 1, most]) if most else ([1, 2],):
        check_attention(rng, heads, kvh, d, 64, [300, 40, 129][:len(q)], q, R.E4M3, half, pad=16)


def test_model_sample(tmp_path):
    """A model's decode loop with sampled tokens, against the 64-bit form on its logits; u = 0 at temperature 0 is the greedy
    token; u outside [0, 1) is refused."""
    import fence_model as M
    from model_files import write_tiny_qwen3
    path = str(tmp_path / "tiny.gguf")
    write_tiny_qwen3(path)
    rng = np.random.default_rng(6)
    with M.Model(path, max_ctx=32) as m:
        tok = 1
        for pos in range(12):
            ptr = m.forward(tok, pos)
            x = m.logits(ptr)
            t, k, p, mp = [(0.8, 0, 0.9, 0.0), (1.5, 7, 1.0, 0.0), (1.0, 0, 1.0, 0.05), (0.0, 0, 1.0, 0.0)][pos % 4]
            u = float(np.float32(rng.random()))
            tok = m.sample(ptr, u, temperature=t, top_k=k, top_p=p, min_p=mp)
            assert tok == R.sample(x, t, k, np.float32(p), np.float32(mp), u)
            if t == 0.0:
                assert tok == m.sample_greedy(ptr)
        for u in (-0.1, 1.0, float("nan")):
            with pytest.raises(F.FenceError):
                m.sample(ptr, u)
