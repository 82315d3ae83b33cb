"""GPU checks of the cache's page tables against a plain host model, and of the
write, attention and page operators used together."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pages(built_library):
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from test_speed_scalesweep_b200 import kv_pages
    return kv_pages


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Model:
    """The tables on the host: lists and loops."""

    def __init__(self, pool, seqs, columns, page):
        self.ref, self.rows, self.lens = [0] * pool, [[] for _ in range(seqs)], [0] * seqs
        self.columns, self.page = columns, page
        self.data = list(range(1000, 1000 + pool))  # what a page holds

    def take(self, n):
        free = [p for p, r in enumerate(self.ref) if r == 0][:n]
        if len(free) < n:
            return None
        for p in free:
            self.ref[p] = 1
        return free

    def extend(self, seqs, more):
        need = [-(-(self.lens[s] + m) // self.page) - len(self.rows[s]) for s, m in zip(seqs, more)]
        got = self.take(sum(need))
        if got is None:
            return None
        slots = []
        for s, m, n in zip(seqs, more, need):
            self.rows[s] += got[:n]
            got = got[n:]
            for t in range(self.lens[s], self.lens[s] + m):
                slots.append(self.rows[s][t // self.page] * self.page + t % self.page)
            self.lens[s] += m
        return slots

    def fork(self, parents, children):
        part = [p for p in parents if self.lens[p] % self.page]
        got = self.take(len(part))
        if got is None:
            return False
        for p, c in zip(parents, children):
            row = list(self.rows[p])
            if self.lens[p] % self.page:
                fresh = got.pop(0)
                self.data[fresh] = self.data[row[-1]]
                row[-1] = fresh
            for q in row[: self.lens[p] // self.page]:
                self.ref[q] += 1
            self.rows[c], self.lens[c] = row, self.lens[p]
        return True

    def free(self, seqs):
        for s in seqs:
            for q in self.rows[s]:
                self.ref[q] -= 1
            self.rows[s], self.lens[s] = [], 0

    def compact(self):
        live = sum(r != 0 for r in self.ref)
        holes = [p for p in range(live) if self.ref[p] == 0]
        high = [p for p in range(live, len(self.ref)) if self.ref[p] != 0]
        to = dict(zip(high, holes))
        for a, b in to.items():
            self.ref[b], self.ref[a], self.data[b] = self.ref[a], 0, self.data[a]
        self.rows = [[to.get(p, p) for p in row] for row in self.rows]

    def compare(self, t):
        rows = [row + [-1] * (self.columns - len(row)) for row in self.rows]
        assert t.block_table.tolist() == rows
        assert t.refcount.tolist() == self.ref
        assert t.seq_lens.tolist() == self.lens


def make(pages, pool, seqs, columns, page=16, layers=2, hkv=1, d=64):
    from test_speed_scalesweep_b200 import kv_cache
    codes, scales = kv_cache.alloc_kv_cache(pool, page, hkv, d, num_layers=layers)
    return pages.NVFP4KVPages.empty(codes, scales, seqs, columns)


def paint(t, model):
    """Give every page bytes of its own, by layer."""
    ids = torch.tensor(model.data, device="cuda")
    for layer in range(t.codes.shape[0]):
        v = ids * 7 + layer * 13
        t.codes[layer] = (v % 251).to(torch.uint8)[:, None, None, None, None]
        t.scales[layer].view(torch.uint8)[:] = (v % 241).to(torch.uint8)[:, None, None, None, None]


def same_data(t, model):
    ids = torch.tensor(model.data, device="cuda")
    live = torch.tensor(model.ref, device="cuda") > 0
    for layer in range(t.codes.shape[0]):
        v = (ids * 7 + layer * 13)[live][:, None, None, None, None]
        assert bool((t.codes[layer][live] == v % 251).all())
        assert bool((t.scales[layer].view(torch.uint8)[live] == v % 241).all())


@pytest.mark.parametrize("seed,pool,seqs,page,hkv,d", [(0, 60, 12, 16, 1, 64), (1, 5000, 40, 32, 3, 128),
                                                       (2, 300, 9, 128, 1, 256), (3, 9000, 300, 16, 1, 64)])
def test_random_use_matches_the_model(pages, seed, pool, seqs, page, hkv, d):
    rng = random.Random(seed)
    columns = 11
    t = make(pages, pool, seqs, columns, page, hkv=hkv, d=d)
    m = Model(pool, seqs, columns, page)
    paint(t, m)
    refused = 0
    for step in range(60):
        op = rng.choice(["extend", "extend", "fork", "free", "compact"])
        if op == "extend":
            who = rng.sample(range(seqs), rng.randint(1, seqs))
            more = [min(rng.choice([0, 1, 5, page, 3 * page + 1]), columns * page - m.lens[s]) for s in who]
            want = m.extend(who, more)
            got = t.extend(i32(who), i32(more), sum(more)).tolist()
            assert got == (want if want is not None else [-1] * sum(more))
            refused += want is None
            if want is None:
                with pytest.raises(RuntimeError, match="not enough"):
                    t.check()
        elif op == "fork":
            empty = [s for s in range(seqs) if m.lens[s] == 0 and not m.rows[s]]
            rng.shuffle(empty)
            empty = empty[: rng.randint(0, len(empty))]
            others = [s for s in range(seqs) if s not in empty]
            if not empty or not others:
                continue
            parents = [rng.choice(others) for _ in empty]
            served = m.fork(parents, empty)
            t.fork(i32(parents), i32(empty))
            if not served:
                refused += 1
                with pytest.raises(RuntimeError, match="not enough"):
                    t.check()
        elif op == "free":
            who = rng.sample(range(seqs), rng.randint(1, max(1, seqs // 3)))
            m.free(who)
            t.free(i32(who + who[:1] if len(who) < seqs else who))
        else:
            m.compact()
            t.compact()
        m.compare(t)
        same_data(t, m)
        t.check()
    if pool == 60:
        assert refused  # the small pool runs out


def test_more_requests_than_threads(pages):
    t, m = make(pages, 20000, 5000, 4, layers=1), Model(20000, 5000, 4, 16)
    who = list(range(0, 5000, 2))
    more = [(7 * s) % 50 for s in who]
    assert t.extend(i32(who), i32(more), sum(more)).tolist() == m.extend(who, more)
    kids = list(range(1, 5000, 2))
    t.fork(i32(who), i32(kids))
    assert m.fork(who, kids)
    m.compare(t)
    t.free(i32(who))
    m.free(who)
    t.compact()
    m.compact()
    m.compare(t)
    t.check()


def test_refused_requests_change_nothing(pages):
    t, m = make(pages, 8, 4, 3), Model(8, 4, 3, 16)
    t.extend(i32([0, 1]), i32([20, 16]), 36)
    m.extend([0, 1], [20, 16])
    m.compare(t)
    for match, call in (
            ("longer", lambda: t.extend(i32([0]), i32([29]), 29)),
            ("index", lambda: t.extend(i32([0, 0]), i32([1, 1]), 2)),
            ("index", lambda: t.extend(i32([0, 4]), i32([1, 1]), 2)),
            ("index", lambda: t.extend(i32([-1]), i32([1]), 1)),
            ("index", lambda: t.extend(i32([2]), i32([-3]), 0)),
            ("index", lambda: t.extend(i32([2]), i32([3]), 5)),
            ("index", lambda: t.extend(i32([0, 1, 2]), i32([1 << 29, 1 << 29, 1 << 29]), 1 << 29)),
            ("not enough", lambda: t.extend(i32([2, 3]), i32([48, 48]), 96)),
            ("index", lambda: t.fork(i32([0]), i32([1]))),
            ("index", lambda: t.fork(i32([0, 0]), i32([2, 2]))),
            ("index", lambda: t.fork(i32([0, 9]), i32([2, 3]))),
            ("index", lambda: t.fork(i32([0]), i32([-5]))),
            ("index", lambda: t.free(i32([7])))):
        call()
        with pytest.raises(RuntimeError, match=match):
            t.check()
        m.compare(t)
    t.extend(i32([]), i32([]), 0)
    t.fork(i32([]), i32([]))
    t.free(i32([]))
    t.check()
    with pytest.raises(ValueError, match="int32"):
        t.free(torch.zeros(1, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError, match="has 4"):
        t.free(i32([0] * 5))
    m.compare(t)


def test_copy_and_graph(pages):
    t, m = make(pages, 40, 6, 5, layers=3), Model(40, 6, 5, 16)
    paint(t, m)
    before = t.codes.clone()
    t.copy(i32([3, 4, -1, 50]), i32([10, 11, 12, 13]))
    before[:, 10], before[:, 11] = before[:, 3], before[:, 4]
    assert torch.equal(t.codes, before)
    who, more, kids, half = i32([0, 1]), i32([33, 5]), i32([4, 5]), i32([0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        slots = t.extend(who, more, 38)
        t.fork(who, kids)
        t.free(half)
        t.compact()
    for _ in range(2):
        m.data = list(range(1000, 1040))
        paint(t, m)
        graph.replay()
        want = m.extend([0, 1], [33, 5])
        m.fork([0, 1], [4, 5])
        m.free([0])
        m.compact()
        assert slots.tolist() == want
        m.compare(t)
        same_data(t, m)
        m.free([1, 4, 5])
        t.free(i32([1, 4, 5]))
    t.check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_serving_run(pages, dtype):
    """Prompts, forks, single tokens, frees and a compaction: every attention result equals the one over
    a cache that was written in one piece, and the cache's rows those of the quantizer."""
    from test_speed_scalesweep_b200 import kv_attention, kv_cache
    hq, hkv, d, page, layers = 8, 2, 128, 16, 2
    g = torch.Generator(device="cuda").manual_seed(3)
    codes, scales = kv_cache.alloc_kv_cache(200, page, hkv, d, num_layers=layers)
    scales.view(torch.uint8).fill_(0x7F)  # NaN wherever nothing was written
    t = pages.NVFP4KVPages.empty(codes, scales, 6, 20)
    table = kv_cache.rotary_cos_sin_cache(400, d)
    mult = torch.tensor([1536 / 9.0, 1536 / 7.0], device="cuda")
    history = {}  # sequence -> qkv of its tokens, by layer

    def step(seqs, more):
        lens = [0 if s not in history else history[s][0].shape[0] for s in seqs]
        slots = t.extend(i32(seqs), i32(more), sum(more))
        pos = torch.cat([torch.arange(n, n + k, device="cuda") for n, k in zip(lens, more)])
        start = torch.tensor([0] + more).cumsum(0).int().cuda()
        result = []
        for layer in range(layers):
            qkv = torch.randn(sum(more), hq + 2 * hkv, d, device="cuda", generator=g).to(dtype)
            q = kv_cache.rotary_scalesweep_mse_nvfp4_kv_write(
                qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:], pos, table, slots, mult, codes[layer],
                scales[layer])
            out = kv_attention.nvfp4_paged_attention(
                q, codes[layer], scales[layer], mult, t.block_table[seqs].contiguous(), t.seq_lens[seqs].contiguous(),
                start, max(more), 320)
            result.append((q, out))
            at = 0
            for s, k in zip(seqs, more):
                old = history.setdefault(s, [qkv[:0]] * layers)
                history[s] = old[:layer] + [torch.cat([old[layer], qkv[at:at + k]])] + old[layer + 1:]
                at += k
        # the same rows over each sequence's own fresh cache
        for layer in range(layers):
            at = 0
            for s, k in zip(seqs, more):
                x = history[s][layer]
                n = x.shape[0]
                c, w = kv_cache.alloc_kv_cache(-(-n // page), page, hkv, d)
                rows = torch.arange(n, device="cuda")
                q = kv_cache.rotary_scalesweep_mse_nvfp4_kv_write(
                    x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], rows, table, rows, mult, c, w)
                assert torch.equal(q[n - k:], result[layer][0][at:at + k])
                out = kv_attention.nvfp4_paged_attention(
                    q[n - k:], c, w, mult, torch.arange(-(-n // page), dtype=torch.int32, device="cuda")[None],
                    i32([n]), i32([0, k]), max(more), 320)
                # other splits, other order of sums: float32 sums and weights rounded to f16 (2^-11 of
                # weights that add up to 1, against values of at most about 5), then one step of the type
                off = (out.float() - result[layer][1][at:at + k].float()).abs().max().item()
                assert off <= 5 * 2.0 ** -10 + 5 * torch.finfo(dtype).eps, off
                at += k
        t.check()

    step([0, 1, 2], [37, 160, 5])
    step([0, 1, 2], [1, 1, 1])
    t.fork(i32([0, 1, 1]), i32([3, 4, 5]))
    for parent, child in ((0, 3), (1, 4), (1, 5)):
        history[child] = list(history[parent])
    step([0, 3, 1, 4, 5], [1, 1, 1, 1, 1])
    t.free(i32([1, 2]))
    del history[1], history[2]
    t.compact()
    used = int((t.refcount > 0).sum())
    assert int((t.refcount[:used] > 0).sum()) == used
    step([0, 3, 4, 5], [1, 60, 2, 1])
    step([2, 1], [100, 1])
    step([0, 1, 2, 3, 4, 5], [1] * 6)


def test_torch_ops_and_a_compiled_layer(pages):
    """The registered ops give the functions' results, in a compiled graph too."""
    from test_speed_scalesweep_b200 import kv_attention, kv_cache, ops  # noqa: F401
    ns = torch.ops.scalesweep_b200
    hq, hkv, d, n = 4, 2, 64, 33
    table, mult = kv_cache.rotary_cos_sin_cache(64, d), torch.tensor([100.0, 120.0], device="cuda")
    qkv = torch.randn(n, hq + 2 * hkv, d, device="cuda", generator=torch.Generator("cuda").manual_seed(0)).bfloat16()
    idx, rows = torch.arange(n, device="cuda"), i32([[2, 0, 1]])

    def layer(x, codes, scales):
        q = ns.rotary_scalesweep_mse_nvfp4_kv_write(x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], idx, table,
                                                    slots, mult, codes, scales, True)
        return ns.nvfp4_paged_attention(q, codes, scales, mult, rows, i32([n]), i32([0, n]), n, n) * 2

    slots = rows[0, idx // 16].long() * 16 + idx % 16
    caches = [kv_cache.alloc_kv_cache(3, 16, hkv, d) for _ in range(2)]
    want = layer(qkv, *caches[0])
    got = torch.compile(layer, backend="aot_eager", fullgraph=True)(qkv, *caches[1])
    assert torch.equal(got, want) and torch.equal(caches[0][0][:, :, :, :1], caches[1][0][:, :, :, :1])
    k, v = ns.nvfp4_kv_gather(*caches[0], mult, slots, torch.float16)
    fk, fv = kv_cache.nvfp4_kv_gather(*caches[1], mult, slots, torch.float16)
    assert torch.equal(k, fk) and torch.equal(v, fv)
