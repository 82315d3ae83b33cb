"""GPU checks of attention over the NVFP4 cache against the formula in 64 bits,
at the lengths, masks and page ends where it can go wrong, with NaN scales in
every row that no query may read."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


@pytest.fixture(scope="module")
def attn(built_library):
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from test_speed_scalesweep_b200 import kv_attention
    return kv_attention


class Batch:
    """A cache whose unused rows are poisoned, and a batch of (keys, queries)."""

    def __init__(self, lens, hq, hkv, d, page, dtype, seed=0, spread=1.0, behind=None, strided=False):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.lens, self.hq, self.hkv, self.d, self.page, self.dtype = lens, hq, hkv, d, page, DT[dtype]
        need = [-(-n // page) for n, _ in lens]
        pages = sum(need) + 3
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))
        self.table = torch.full((len(lens), max(need + [1]) + 2), -1, dtype=torch.int32)
        shape = (pages, 2, hkv, page)
        codes = torch.randint(0, 256, shape + (d // 2,), dtype=torch.uint8, device="cuda", generator=g)
        # scales over a range of 2^7, subnormal E4M3 among them
        raw = torch.randint(1, 70, shape + (d // 16,), dtype=torch.uint8, device="cuda", generator=g)
        at = 0
        for i, (n, _) in enumerate(lens):
            ids = order[at:at + need[i]]
            self.table[i, :need[i]] = ids.int()
            at += need[i]
            if n % page:
                codes[ids[-1], :, :, n % page:] = 0x77
                raw[ids[-1], :, :, n % page:] = 0x7F  # NaN
            for col in range((behind or {}).get(i, 0) // page):  # pages that a window left behind
                codes[ids[col]], raw[ids[col]] = 0x77, 0x7F
                self.table[i, col] = -1 if col % 2 else pages + 7
        for p in order[at:].tolist():
            codes[p], raw[p] = 0x77, 0x7F
        self.codes, self.raw, self.scales = codes, raw, raw.view(torch.float8_e4m3fn)
        self.table_cpu, self.table = self.table, self.table.cuda()
        t = sum(q for _, q in lens)
        width = hq + (2 * hkv if strided else 0)
        self.q = (spread * torch.randn(t, width, d, device="cuda", generator=g)).to(self.dtype)[:, :hq]
        self.mult = torch.tensor([9.0, 3.5], device="cuda")
        self.seq_lens = torch.tensor([n for n, _ in lens], dtype=torch.int32, device="cuda")
        starts = [0]
        for _, q in lens:
            starts.append(starts[-1] + q)
        self.start = torch.tensor(starts, dtype=torch.int32, device="cuda")
        self.max_q, self.max_s = max(q for _, q in lens), max(max(n for n, _ in lens), 1)

    def call(self, attn, **kw):
        return attn.nvfp4_paged_attention(self.q, self.codes, self.scales, self.mult, self.table,
                                          self.seq_lens, self.start, max(self.max_q, 1), self.max_s, **kw)

    def dense(self, i, h, side):
        n = self.lens[i][0]
        ids = self.table_cpu[i, : -(-n // self.page)].long()
        present = (ids >= 0) & (ids < self.codes.shape[0])
        ids = torch.where(present, ids, 0).cuda()
        c = self.codes[ids, side, h].reshape(-1, self.d // 2)[:n]
        s = self.raw[ids, side, h].reshape(-1, self.d // 16)[:n].contiguous().view(torch.float8_e4m3fn).double()
        value = torch.tensor(E2M1 + tuple(-e for e in E2M1), dtype=torch.float64, device="cuda")
        x = value[torch.stack([c & 15, c >> 4], -1).long()].reshape(n, -1, 16) * s[..., None]
        return x.reshape(n, self.d) / self.mult[side].double(), present.repeat_interleave(self.page)[:n].cuda()

    def check(self, out, lse=None, causal=True, window=None, scale=None):
        scale = self.d ** -0.5 if scale is None else scale
        at = 0
        for i, (n, m) in enumerate(self.lens):
            for h in range(self.hkv):
                if n:
                    k, there = self.dense(i, h, 0)
                    v, _ = self.dense(i, h, 1)
                g = self.hq // self.hkv
                q = self.q[at:at + m, h * g:(h + 1) * g].double()
                got = out[at:at + m, h * g:(h + 1) * g].double()
                pos = torch.arange(m, device="cuda")[:, None] + n - m
                key = torch.arange(n, device="cuda")[None]
                keep = torch.ones(m, n, dtype=torch.bool, device="cuda")
                if n:
                    keep &= there[None]
                if causal:
                    keep &= key <= pos
                if window is not None:
                    keep &= key >= pos - window
                for j in range(g):
                    if n == 0:
                        assert bool((got[:, j] == 0).all())
                        continue
                    k0 = torch.where(there[:, None], k, 0)
                    v0 = torch.where(there[:, None], v, 0)
                    logit = (q[:, j] @ k0.T * scale).masked_fill(~keep, -math.inf)
                    none = ~keep.any(1)
                    p = torch.softmax(logit, -1)
                    p[none] = 0
                    want, weight = p @ v0, p @ v0.abs()
                    # The score of a key is off by at most D half steps of 2^-23 (products of 16-bit
                    # floats are exact; the tensor cores may cut instead of round) of what its terms
                    # could add up to, which moves a weight and the weights' sum by as much each.
                    # A weight is rounded to f16: 2^-11, or 2^-34 of the largest where it is tiny.
                    # The result is rounded once to its type: half a step, which for a subnormal of
                    # the type is half its smallest one.
                    reach = scale * q[:, j].abs().amax(1, keepdim=True) * k0.abs().sum(1).amax()
                    logit_off = self.d * 2.0 ** -23 * abs(reach) + 2.0 ** -20
                    f = torch.finfo(self.dtype)
                    tol = (f.eps / 2 * want.abs().clamp(min=f.smallest_normal)
                           + (2.0 ** -11 + 2 * logit_off) * weight + n * 2.0 ** -34 * v0.abs().amax())
                    off = (got[:, j] - want).abs()
                    bad = ~(off <= tol + 1e-300)
                    assert not bool(bad.any()), (i, h, j, bad.nonzero()[0].tolist(), off[bad][0].item(), tol[bad][0].item())
                    if lse is not None:
                        mine = lse[at:at + m, h * g + j].double()
                        ref = torch.logsumexp(logit, -1)
                        assert bool((mine[none] == -math.inf).all())
                        # the sum of weights is off as they are; a float32 result near |lse|
                        lim = logit_off[:, 0] + 2.0 ** -18 + ref.abs() * 2.0 ** -22
                        ok = (mine - ref).abs() <= lim
                        assert bool(ok[~none].all())
            at += m


SHORT = [  # (lengths, hq, hkv, d, page)
    ([(1, 1)], 1, 1, 64, 16), ([(1024, 1)], 32, 8, 128, 16), ([(17, 1), (1, 1), (333, 1), (2048, 1)], 8, 2, 128, 32),
    ([(31, 1), (32, 1), (33, 1), (0, 1), (129, 1)], 6, 6, 64, 16), ([(700, 2), (90, 5), (5, 5)], 10, 2, 128, 64),
    ([(515, 1), (128, 3)], 12, 3, 256, 16), ([(4000, 8), (77, 1)], 8, 1, 64, 128), ([(260, 4), (3, 4)], 16, 2, 256, 32)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("lens,hq,hkv,d,page", SHORT)
def test_short_queries(attn, lens, hq, hkv, d, page, dtype):
    b = Batch(lens, hq, hkv, d, page, dtype, seed=len(lens) + d, spread=1.5)
    out, lse = b.call(attn, return_lse=True)
    b.check(out, lse)


LONG = [
    ([(128, 128)], 4, 1, 128, 16), ([(300, 300), (1, 1), (129, 65)], 8, 2, 128, 32), ([(1000, 37), (64, 64)], 6, 2, 64, 64),
    ([(513, 200)], 5, 1, 256, 16), ([(2000, 129), (255, 255), (40, 1), (0, 3), (3, 7)], 8, 8, 64, 16), ([(777, 777)], 3, 3, 128, 128),
    ([(1537, 65)], 8, 8, 256, 64)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("lens,hq,hkv,d,page", LONG)
def test_long_queries(attn, lens, hq, hkv, d, page, dtype):
    b = Batch(lens, hq, hkv, d, page, dtype, seed=len(lens) + d, spread=1.5, strided=True)
    out, lse = b.call(attn, return_lse=True)
    b.check(out, lse)


@pytest.mark.parametrize("lens", [[(900, 1), (70, 1), (3, 1)], [(900, 9), (64, 64), (400, 130)], [(1500, 1), (1500, 600)]])
@pytest.mark.parametrize("window", [0, 1, 31, 100, 4000])
def test_windows_and_pages_left_behind(attn, lens, window):
    # pages that lie before every query's window are gone from the table
    behind = {i: max(0, n - m - window) for i, (n, m) in enumerate(lens)}
    b = Batch(lens, 8, 2, 128, 16, "bf16", seed=window, behind=behind)
    out, lse = b.call(attn, window=window, return_lse=True)
    b.check(out, lse, window=window)


@pytest.mark.parametrize("lens", [[(513, 1), (40, 3)], [(513, 100), (40, 40), (7, 30)]])
def test_without_causal_order_and_own_scale(attn, lens):
    b = Batch(lens, 4, 2, 64, 32, "f16", seed=5)
    b.check(b.call(attn, causal=False, softmax_scale=0.3), causal=False, scale=0.3)
    b.check(b.call(attn, softmax_scale=-0.2), scale=-0.2)
    b.check(b.call(attn, softmax_scale=0.0), scale=0.0)


@pytest.mark.parametrize("lens", [[(2592, 394), (9, 1)], [(1536, 1), (724, 4), (5000, 2)]])
@pytest.mark.parametrize("window", [3, 211])
def test_window_without_causal_order(attn, lens, window):
    # such a query sees every key from window positions before it to the last one
    b = Batch(lens, 8, 2, 64, 16, "bf16", seed=window)
    b.check(b.call(attn, causal=False, window=window), causal=False, window=window)


@pytest.mark.parametrize("m", [1, 140])
def test_peaked_and_flat_scores(attn, m):
    # one key far above the rest, and rows of very different sizes
    b = Batch([(3000, m)], 4, 1, 128, 16, "bf16", seed=8)
    b.q.mul_(torch.logspace(-30, 1.3, 4, device="cuda").bfloat16()[None, :, None])
    b.check(b.call(attn))


@pytest.mark.parametrize("m", [1, 7, 200])
def test_rows_behind_the_last_sequence_and_output_strides(attn, m):
    b = Batch([(300, m), (50, m if m < 50 else 50)], 4, 2, 64, 16, "bf16", seed=2)
    t = b.q.shape[0]
    wide = torch.full((t + 5, 6, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    q = torch.cat([b.q, torch.full((5, 4, 64), float("nan"), dtype=torch.bfloat16, device="cuda")])
    got = attn.nvfp4_paged_attention(q, b.codes, b.scales, b.mult, b.table, b.seq_lens, b.start, b.max_q,
                                     b.max_s, out=wide[:, 1:5])
    assert got.data_ptr() == wide[:, 1:5].data_ptr()
    b.check(wide[:t, 1:5])
    assert bool((wide[t:] == 7).all()) and bool((wide[:, 0] == 7).all()) and bool((wide[:, 5] == 7).all())


@pytest.mark.parametrize("lens", [[(4096, 1)] * 3, [(2048, 300), (4096, 1)]])
def test_deterministic_streams_graphs_and_two_at_once(attn, lens):
    b = Batch(lens, 8, 2, 128, 16, "bf16", seed=4)
    c = Batch(lens, 8, 2, 128, 16, "bf16", seed=6)
    want, other = b.call(attn), c.call(attn)
    assert torch.equal(want, b.call(attn))
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    graphs = []
    for batch, s in ((b, s1), (c, s2)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = batch.call(attn)
        graphs.append((g, out, s))
    for _ in range(3):
        for g, _, s in graphs:
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], want) and torch.equal(graphs[1][1], other)
    b.q.copy_(c.q)
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], b.call(attn))


def test_pages_past_32_bits(attn):
    """A cache of more than 2^32 bytes of codes: the last pages answer as the first do."""
    from test_speed_scalesweep_b200 import kv_cache
    b = Batch([(200, 1), (100, 70)], 8, 8, 128, 128, "bf16", seed=1)
    pages = (1 << 32) // (2 * 8 * 128 * 64) + b.codes.shape[0] + 1
    codes, scales = kv_cache.alloc_kv_cache(pages, 128, 8, 128)
    shift = pages - b.codes.shape[0]
    codes[shift:] = b.codes
    scales.view(torch.uint8)[shift:] = b.raw
    table = torch.where(b.table >= 0, b.table + shift, b.table)
    got = attn.nvfp4_paged_attention(b.q, codes, scales, b.mult, table, b.seq_lens, b.start, b.max_q, b.max_s)
    assert torch.equal(got, b.call(attn))


def test_status_stays_clear(attn):
    b = Batch([(300, 1), (300, 200)], 4, 2, 128, 16, "bf16")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    b.call(attn, status=status)
    assert status.item() == 0


@pytest.mark.parametrize("lens", [[(9000, 1)], [(9000, 1), (500, 1)], [(9000, 40)], [(5000, 300), (9000, 1)]])
def test_bounds_smaller_than_the_batch_stay_in_bounds(attn, lens):
    """Lengths past the bounds are passed over; the queries within them still look at the keys within them."""
    b = Batch(lens, 4, 1, 128, 16, "bf16", seed=3)
    guard = torch.full((b.q.shape[0], 4, 128), 5.0, dtype=torch.bfloat16, device="cuda")
    for max_q, max_s in ((b.max_q, 700), (1, 9000), (1, 1)):
        out = attn.nvfp4_paged_attention(b.q, b.codes, b.scales, b.mult, b.table, b.seq_lens, b.start, max_q,
                                         max_s, out=guard.clone())
        assert bool(out[0].isfinite().all()) and bool((out[0] != 5).any())
    b.check(b.call(attn))


@pytest.mark.parametrize("lens", [[(4096, 1)] * 3, [(2048, 300), (4096, 1), (64, 1)], [(5000, 1)]])
def test_reads_what_the_launch_before_wrote(attn, lens):
    """Launches overlap their predecessors' ends: inputs written just before a call, into lines that the call
    before it has read, are the ones that it sees."""
    b, c = Batch(lens, 8, 2, 128, 16, "bf16", seed=4), Batch(lens, 8, 2, 128, 16, "bf16", seed=6)
    fewer = [(n - 1, q) for n, q in lens]
    c.seq_lens.copy_(torch.tensor([n for n, _ in fewer], dtype=torch.int32))
    inputs = [[t.clone() for t in (x.q, x.codes, x.raw, x.table, x.seq_lens, x.mult)] for x in (b, c)]
    inputs[1][5].mul_(2)
    mine = (b.q, b.codes, b.raw, b.table, b.seq_lens, b.mult)

    def load(which):
        for dst, src in zip(mine, inputs[which]):
            dst.copy_(src)
    want = []
    for which in (0, 1):
        load(which)
        torch.cuda.synchronize()
        want.append(b.call(attn))
        torch.cuda.synchronize()
    got = []
    for i in range(24):
        load(i % 2)
        got.append(b.call(attn))
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        assert torch.equal(out, want[i % 2]), i


def test_two_host_threads(attn):
    """Calls of two threads through the C interface, which holds no lock: a long sequence and a batch of short
    ones use one kernel with different launch settings."""
    import ctypes
    import threading

    from test_speed_scalesweep_b200 import _lib
    lib = _lib.lib()
    jobs = []
    for lens in ([(60000, 1)], [(900, 1)] * 4):
        b = Batch(lens, 8, 8, 128, 16, "bf16", seed=5)
        want = b.call(attn)
        out = torch.empty_like(want)
        cache = _lib.KVCache(codes=b.codes.data_ptr(), scales=b.raw.data_ptr(), codes_page_stride=b.codes.stride(0),
                             scales_page_stride=b.raw.stride(0), input_scale=b.mult.data_ptr(),
                             num_pages=b.codes.shape[0], page_size=16, kv_heads=8, head_size=128)
        args = _lib.KVAttention(block_table=b.table.data_ptr(), block_table_stride=b.table.stride(0),
                                seq_lens=b.seq_lens.data_ptr(), query_start=b.start.data_ptr(), tokens=len(lens),
                                seqs=len(lens), block_table_columns=b.table.shape[1], q_heads=8, max_query_len=1,
                                max_seq_len=b.max_s, causal=1, window=-1, softmax_scale=128 ** -0.5)
        q, o = _lib.KVHeads(b.q.data_ptr(), 8 * 128, 128), _lib.KVHeads(out.data_ptr(), 8 * 128, 128)
        need = lib.ssw_nvfp4_paged_attention_workspace_bytes(ctypes.byref(cache), ctypes.byref(args), 0)
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
        jobs.append((b, want, out, (ctypes.byref(cache), ctypes.byref(args), 0, ctypes.byref(q), ctypes.byref(o),
                                    ws.data_ptr(), need, torch.cuda.Stream().cuda_stream), ws))
    torch.cuda.synchronize()
    bad = []

    def run(call):
        for _ in range(400):
            if lib.ssw_nvfp4_paged_attention(*call) != 0:
                bad.append(lib.ssw_last_error())
    threads = [threading.Thread(target=run, args=(j[3],)) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not bad, bad[:1]
    for _, want, out, _, _ in jobs:
        assert torch.equal(out, want)
