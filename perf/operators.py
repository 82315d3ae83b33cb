"""Measured cases of the 4-bit KV cache operators.

Three operators, as a serving program calls them between the qkv and the output projection of a decoder layer:

* ``write``:  rotary positions on the query and key heads of a qkv projection's output, and the scale-sweep NVFP4
  quantization of the keys and values into the pages of a cache; the pass reads the written rows back as values.
* ``attend``: attention over such a cache: single tokens, chunks of prompts, and batches that mix both.
* ``pages``:  forking sequences, and freeing, compacting and extending them, over all layers of a cache.

``own = False`` computes them from elementary torch operations; ``own = True`` calls the package.
"""
import math

import numpy as np
import torch

own = False

# Lowest code whose distance from the base scale's code the sweep tries, and how many it tries.
LOWER, WINDOW = -3, 11
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ---- cases -------------------------------------------------------------------------------------------------------
def listed():
    write = dict(op="write", dtype="bf16", hq=32, hkv=8, d=128, rot=128, neox=True, page=16, scaling="llama3")
    attend = dict(op="attend", dtype="bf16", hq=32, hkv=8, d=128, page=16, window=0)
    pages = dict(op="pages", hkv=8, d=128, page=16)
    return [
        # one token of one sequence: the latency of a decode step's write
        dict(write, name="write 1 token", tokens=1, start=1000, padding=0),
        # a decode batch of an interleaved model that rotates half of each head
        dict(write, name="write 256 tokens interleaved", tokens=256, start=30000, padding=0, hq=16, hkv=16, rot=64, neox=False, scaling="none", page=32),
        # a padded odd batch in fp16, small heads, far positions
        dict(write, name="write 1999 tokens fp16", tokens=1999, start=120000, padding=49, dtype="fp16", hq=24, hkv=6, d=64, rot=64, scaling="yarn", page=64),
        # a prompt chunk
        dict(write, name="write 8192 tokens", tokens=8192, start=4096, padding=0),
        # one sequence's decode step
        dict(attend, name="attend decode 1 x 1024", seqs=1, queries=1, context=1024, ragged=False),
        # a decode batch of uneven lengths
        dict(attend, name="attend decode 64 ragged", seqs=64, queries=1, context=8192, ragged=True),
        # one very long sequence
        dict(attend, name="attend decode 1 x 131072", seqs=1, queries=1, context=131072, ragged=False),
        # prompts and single tokens in one batch, fp16, small heads, a sliding window
        dict(attend, name="attend mixed fp16 window", seqs=24, queries=333, context=3001, ragged=True, dtype="fp16", hq=24, hkv=6, d=64, page=64, window=1024),
        # a prompt chunk over its cached beginning
        dict(attend, name="attend prefill 4096 of 16384", seqs=1, queries=4096, context=16384, ragged=False),
        # parallel sampling: each prompt forked four ways
        dict(pages, name="pages fork 8 x 4", kind="fork", layers=2, seqs=8, fan=4, context=777, pool=2048),
        dict(pages, name="pages fork 64 x 4", kind="fork", layers=32, seqs=64, fan=4, context=300, pool=2048),
        # finished sequences leave holes, the pool is compacted, new ones come in
        dict(pages, name="pages compact 4096", kind="compact", layers=8, seqs=96, fan=1, context=600, pool=4096),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    dtype = rng.choice(["bf16", "fp16"])
    d = rng.choice([64, 128, 128, 256])
    hkv = rng.choice([1, 2, 4, 6, 8])
    group = rng.choice([1, 2, 3, 4, 5, 8])
    page = rng.choice([16, 32, 64, 128])
    op = rng.choice(["write", "attend", "attend", "pages"])
    if op == "write":
        tokens = _spread(rng, 1, 8192 * 6144 // (hkv * (group + 2) * d) if hkv * (group + 2) * d > 6144 else 8192)
        return dict(op=op, dtype=dtype, hq=hkv * group, hkv=hkv, d=d, rot=16 * rng.randint(1, d // 16), neox=rng.random() < 0.6, page=page,
                    scaling=rng.choice(["none", "linear", "llama3", "yarn"]), tokens=tokens, start=rng.randint(0, 120000), padding=rng.randint(0, tokens // 8))
    if op == "attend":
        hq = hkv * group
        context = _spread(rng, 1, 32768)
        if rng.random() < 0.5:
            queries = 1 if rng.random() < 0.7 else rng.randint(2, 8)
            # no more keys than the largest decode batch reads, no more scores than the largest prompt's
            seqs = _spread(rng, 1, max(1, min(128, 64 * 8192 * 8 * 128 // (context * hkv * d * 2), 1 << 30 // max(1, context * queries * hq))))
        else:
            queries = _spread(rng, 9, 4096)
            # a prompt's scores, and its products, are no more than the largest listed prompt's
            most = (1 << 31) * 128 // max(d, 128)
            seqs = rng.randint(1, max(1, min(16, most // (context * queries * hq), (1 << 30) // (context * hkv * d))))
            queries = max(9, min(queries, most // (context * seqs * hq)))
        return dict(op=op, dtype=dtype, hq=hq, hkv=hkv, d=d, page=page, window=rng.choice([0, 0, 0, _spread(rng, 1, 4096)]), seqs=seqs, queries=queries,
                    context=max(context, 1), ragged=rng.random() < 0.6)
    kind = rng.choice(["fork", "compact"])
    layers = rng.choice([1, 2, 4, 8])
    page = rng.choice([16, 32])
    context = rng.randint(1, 700)
    each = -(-context // page) + 1
    pool = max(64, min(4096, (1 << 29) // (layers * hkv * page * d)))
    fan = rng.randint(1, 8) if kind == "fork" else 1
    moved = 2 * layers * 2 * hkv * page * (d // 2 + d // 16)  # bytes of a page copied
    seqs = rng.randint(1, max(1, min(96, pool // (each + fan), 250_000_000 // (moved * fan))))
    return dict(op="pages", hkv=hkv, d=d, page=page, kind=kind, layers=layers, seqs=seqs, fan=fan, context=context, pool=max(pool, seqs * (each + fan)))


def _type(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float16


def _lengths(case):
    """Sequence lengths and query lengths, the same for every seed: the work does not hang on it."""
    r = np.random.RandomState(case["context"] * 31 + case["seqs"])
    n, c, q = case["seqs"], case["context"], min(case["queries"], case["context"])
    if not case["ragged"]:
        return [c] * n, [q] * n
    seq = [max(1, int(c * u)) for u in r.uniform(0.02, 1.0, n)]
    seq[r.randint(n)] = c
    # every third sequence of a batch of prompts decodes a single token
    qry = [min(s, 1 if q > 8 and i % 3 == 1 else max(1, int(q * u)) if q > 8 else q) for i, (s, u) in enumerate(zip(seq, r.uniform(0.1, 1.0, n)))]
    return seq, qry


def _visible(case):
    """(query, key) pairs a head looks at, and keys that a kv head's cache has to give."""
    w, pairs, keys = case["window"], 0, 0
    for s, q in zip(*_lengths(case)):
        first = s - q  # position of the first query
        sees = np.arange(first + 1, s + 1)
        pairs += int(np.minimum(sees, w + 1).sum()) if w else int(sees.sum())
        keys += min(s, w + q) if w else s
    return pairs, keys


def _page_lengths(case):
    r = np.random.RandomState(case["context"] + 7 * case["seqs"])
    return [max(1, int(case["context"] * u)) for u in r.uniform(0.4, 1.0, case["seqs"])]


def work(case):
    if case["op"] == "write":
        t, live, d = case["tokens"], case["tokens"] - case["padding"], case["d"]
        values = 2 * case["hkv"] * d
        byt = t * (2 * case["hq"] * d * 2 + 4 * case["rot"] + 16) + live * values * (2 + 9 / 16 + 2)
        # per quantized element: 3 operations for each of 11 candidates, and 2; 3 for each rotated one
        return {"bytes": byt, "flops": live * values * 35 + 3 * t * (case["hq"] + case["hkv"]) * case["rot"]}
    if case["op"] == "attend":
        pairs, keys = _visible(case)
        rows = sum(_lengths(case)[1])
        return {"bytes": keys * case["hkv"] * case["d"] * 2 * 9 / 16 + 2 * 2 * rows * case["hq"] * case["d"], "flops": 4 * case["d"] * case["hq"] * pairs}
    size = case["layers"] * 2 * case["hkv"] * case["page"] * (case["d"] // 2 + case["d"] // 16)
    lens, p = _page_lengths(case), case["page"]
    if case["kind"] == "fork":
        moved = case["fan"] * sum(1 for n in lens if n % p)
        return {"bytes": 2 * size * moved + 8 * case["fan"] * sum(-(-n // p) for n in lens) + 4 * case["pool"], "flops": moved}
    gone = sum(-(-n // p) for n in lens[::4])
    moved = gone // 2  # about: what lies above the live pages moves into the holes
    return {"bytes": 2 * size * moved + 4 * case["pool"] * 2, "flops": moved}


# ---- inputs ------------------------------------------------------------------------------------------------------
def _table(positions, rot, scaling):
    """cos and sin of position x frequency, side by side, float32 [positions, rot]; formed in 64 bits."""
    i = torch.arange(0, rot, 2, dtype=torch.float64, device="cuda")
    freq = 500000.0 ** (-i / rot)
    mult = 1.0
    if scaling == "linear":
        freq = freq / 8.0
    elif scaling == "llama3":  # factor 8, low 1, high 4, 8192 positions
        wave = 2 * math.pi / freq
        smooth = ((8192.0 / wave) - 1.0) / 3.0
        mid = (1 - smooth) * freq / 8.0 + smooth * freq
        freq = torch.where(wave > 8192.0, freq / 8.0, torch.where(wave < 2048.0, freq, mid))
    elif scaling == "yarn":  # factor 4, beta 32 and 1, 32768 positions
        def at(turns):
            return rot * math.log(32768.0 / (turns * 2 * math.pi)) / (2 * math.log(500000.0))
        low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
        ramp = ((i / 2 - low) / max(high - low, 0.001)).clamp(0, 1)
        freq = freq / 4.0 * ramp + freq * (1 - ramp)
        mult = 0.1 * math.log(4.0) + 1.0
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * freq
    return torch.cat([angle.cos() * mult, angle.sin() * mult], -1).float()


def _cache(pages, hkv, page, d, gen, layers=None):
    """A cache of keys and values near a normal distribution: scales about amax / 6 of their blocks, codes that fill them."""
    shape = ((layers,) if layers else ()) + (pages, 2, hkv, page)
    codes = torch.randint(0, 256, shape + (d // 2,), dtype=torch.uint8, device="cuda", generator=gen)
    scales = (40.0 + 40.0 * torch.rand(shape + (d // 16,), device="cuda", generator=gen)).to(torch.float8_e4m3fn)
    return codes, scales


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    host = np.random.RandomState(seed % (1 << 31))
    s = dict(case)
    if case["op"] == "write":
        t, d, hq, hkv, p = case["tokens"], case["d"], case["hq"], case["hkv"], case["page"]
        qkv = torch.randn(t, hq + 2 * hkv, d, device="cuda", generator=gen)
        # a few strong channels, as keys have them
        qkv = (qkv * torch.exp(0.5 * torch.randn(hq + 2 * hkv, d, device="cuda", generator=gen))).to(_type(case))
        live = t - case["padding"]
        pages = -(-live // p) + 3
        order = torch.from_numpy(host.permutation(pages)).cuda()
        tok = torch.arange(live, device="cuda")
        slots = torch.full((t,), -1, dtype=torch.int64, device="cuda")
        slots[:live] = order[tok // p] * p + tok % p
        pos = torch.zeros(t, dtype=torch.int64, device="cuda")
        pos[:live] = case["start"] + tok
        codes, scales = _cache(pages, hkv, p, d, gen)
        s.update(q=qkv[:, :hq], k=qkv[:, hq:hq + hkv], v=qkv[:, hq + hkv:], positions=pos, slots=slots, codes=codes, scales=scales,
                 table=_table(case["start"] + t, case["rot"], case["scaling"]), mult=1536.0 / torch.tensor([23.17, 21.91], device="cuda"))  # the maxima, averaged over calibration batches
    elif case["op"] == "attend":
        seq, qry = _lengths(case)
        d, p = case["d"], case["page"]
        need = [-(-n // p) for n in seq]
        pages = sum(need) + 2
        order = host.permutation(pages)
        table = np.full((len(seq), max(need) + 1), -1, np.int32)
        at = 0
        for i, n in enumerate(need):
            table[i, :n] = order[at:at + n]
            at += n
        codes, scales = _cache(pages, case["hkv"], p, d, gen)
        q = 1.5 * torch.randn(sum(qry), case["hq"], d, device="cuda", generator=gen)
        start = np.concatenate([[0], np.cumsum(qry)]).astype(np.int32)
        # a value is code x scale / multiplier: the random codes' mean square is 9, the scales' about 60^2, so that keys are near 1
        s.update(q=q.to(_type(case)), codes=codes, scales=scales, mult=torch.tensor([180.0, 180.0], device="cuda"), block_table=torch.from_numpy(table).cuda(),
                 seq_lens=torch.tensor(seq, dtype=torch.int32, device="cuda"), start=torch.from_numpy(start).cuda(), max_q=max(qry), max_s=max(seq))
    else:
        lens, p = _page_lengths(case), case["page"]
        need = [-(-n // p) for n in lens]
        order = host.permutation(sum(need) if case["kind"] == "compact" else case["pool"])
        total = case["seqs"] * (1 + (case["fan"] if case["kind"] == "fork" else 0))
        table = np.full((total, max(need) + 1), -1, np.int32)
        count = np.zeros(case["pool"], np.int32)
        at = 0
        for i, n in enumerate(need):
            table[i, :n] = order[at:at + n]
            at += n
            count[table[i, :n]] = 1
        codes, scales = _cache(case["pool"], case["hkv"], p, case["d"], gen, case["layers"])
        seq_lens = np.zeros(total, np.int32)
        seq_lens[:len(lens)] = lens
        s.update(codes=codes, scales=scales, block_table=torch.from_numpy(table).cuda(), refcount=torch.from_numpy(count).cuda(), seq_lens=torch.from_numpy(seq_lens).cuda())
        if case["kind"] == "fork":
            s.update(parents=torch.arange(case["seqs"], dtype=torch.int32, device="cuda").repeat_interleave(case["fan"]),
                     children=case["seqs"] + torch.from_numpy(host.permutation(total - case["seqs"]).astype(np.int32)).cuda())
        else:
            drop = np.arange(0, case["seqs"], 4).astype(np.int32)
            back = [lens[i] for i in drop]
            s.update(drop=torch.from_numpy(drop).cuda(), back=torch.tensor(back, dtype=torch.int32, device="cuda"), total=sum(back))
    return s


# ---- the plain forms -----------------------------------------------------------------------------------------------
def _rotate(x, table, positions, rot, neox):
    """Rotary positions in 32 bits, rounded once to x's type."""
    row = table[positions][:, None]
    c, s = row[..., : rot // 2], row[..., rot // 2:]
    y = x.float()
    a, b = (y[..., : rot // 2], y[..., rot // 2: rot]) if neox else (y[..., 0:rot:2], y[..., 1:rot:2])
    oa, ob = a * c - b * s, b * c + a * s
    turned = torch.cat([oa, ob], -1) if neox else torch.stack([oa, ob], -1).flatten(-2)
    return torch.cat([turned, y[..., rot:]], -1).to(x.dtype)


def _nearest(a):
    """Code of the nearest E2M1 value of |a|; ties go to the even code."""
    return (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)


def _quantize(x, mult):
    """Scale sweep of blocks of 16: (codes [.., n/2], scales [.., n/16]); the lowest of the best candidates wins."""
    value = torch.tensor(E2M1, device=x.device)
    v = x.float() * mult
    blocks = v.unflatten(-1, (-1, 16))
    base = (blocks.abs().amax(-1) * torch.tensor(1.0 / 6.0, device=x.device)).clamp(max=448.0).to(torch.float8_e4m3fn).view(torch.uint8)
    raw = (base[..., None].int() + torch.arange(LOWER, LOWER + WINDOW, device=x.device)).clamp(1, 126).to(torch.uint8)
    scale = raw.view(torch.float8_e4m3fn).float()
    y = (blocks[..., None, :] * (1.0 / scale)[..., None]).abs()
    # the candidates' errors lie close together: squares are summed in 64 bits
    off = (value[_nearest(y).int()] - y).double().square().sum(-1) * scale.double().square()
    place = torch.arange(WINDOW, device=x.device)
    first = torch.where(off == off.amin(-1, keepdim=True), place, WINDOW).amin(-1, keepdim=True)
    best = raw.gather(-1, first)
    y = blocks * (1.0 / best.view(torch.float8_e4m3fn).float())
    code = _nearest(y.abs()) + 8 * torch.signbit(y).to(torch.uint8)
    code = code.flatten(-2)
    return code[..., 0::2] + 16 * code[..., 1::2], best[..., 0].view(torch.float8_e4m3fn)


def _values(codes, scales, mult):
    """The values that codes and scales stand for, in 32 bits."""
    signed = torch.tensor(E2M1 + tuple(-e for e in E2M1), device=codes.device)
    v = torch.stack([signed[(codes & 15).int()], signed[(codes >> 4).int()]], -1).flatten(-2)
    return (v.unflatten(-1, (-1, 16)) * scales.float()[..., None]).flatten(-2) / mult


def _plain_write(s):
    q = _rotate(s["q"], s["table"], s["positions"], s["rot"], s["neox"])
    k = _rotate(s["k"], s["table"], s["positions"], s["rot"], s["neox"])
    live = s["slots"] >= 0
    at = s["slots"][live]
    page, row = at // s["page"], at % s["page"]
    back = []
    for side, x in ((0, k), (1, s["v"])):
        codes, scales = _quantize(x[live], s["mult"][side])
        s["codes"][page, side, :, row] = codes
        s["scales"].view(torch.uint8)[page, side, :, row] = scales.view(torch.uint8)
        full = torch.zeros(x.shape, dtype=x.dtype, device=x.device)
        full[live] = _values(s["codes"][page, side, :, row], s["scales"].view(torch.uint8)[page, side, :, row].view(torch.float8_e4m3fn), s["mult"][side]).to(x.dtype)
        back.append(full)
    return {"query": q, "key": back[0], "value": back[1]}


def _plain_attend(s):
    n, maxq, hkv, d = s["seq_lens"].numel(), s["max_q"], s["hkv"], s["d"]
    group = s["hq"] // hkv
    need = -(-s["max_s"] // s["page"])
    at = s["block_table"][:, :need].clamp(min=0).long()
    # [n, pages, 2, hkv, page, .] -> [2, n, hkv, keys, .]
    kc = s["codes"][at].permute(2, 0, 3, 1, 4, 5).flatten(3, 4)
    sc = s["scales"].view(torch.uint8)[at].permute(2, 0, 3, 1, 4, 5).flatten(3, 4).contiguous().view(torch.float8_e4m3fn)
    k, v = _values(kc[0], sc[0], s["mult"][0]), _values(kc[1], sc[1], s["mult"][1])
    lens = (s["start"][1:] - s["start"][:-1])[:, None]
    i = torch.arange(maxq, device=k.device)[None]
    row = (s["start"][:-1, None] + i).clamp(max=s["q"].shape[0] - 1).long()
    q = s["q"][row].float().view(n, maxq, hkv, group, d).permute(0, 2, 3, 1, 4).reshape(n, hkv, group * maxq, d)
    score = (q @ k.transpose(-1, -2)).mul_(d ** -0.5).view(n, hkv, group, maxq, -1)
    pos = (s["seq_lens"][:, None] - lens + i)[:, None, None, :, None]
    key = torch.arange(score.shape[-1], device=k.device)
    hidden = key > pos
    if s["window"]:
        hidden = hidden | (key < pos - s["window"])
    score.masked_fill_(hidden, -math.inf)
    score.sub_(score.amax(-1, keepdim=True)).exp_()
    total = score.sum(-1)
    o = (score.view(n, hkv, group * maxq, -1) @ v).view(n, hkv, group, maxq, d) / total[..., None]
    o = o.permute(0, 3, 1, 2, 4).reshape(n, maxq, hkv * group, d)
    return o[(i < lens)].to(s["q"].dtype)


def _plain_fork(s):
    p = s["page"]
    parents, children = s["parents"].long(), s["children"].long()
    lens = s["seq_lens"][parents]
    rows = s["block_table"][parents]
    column = torch.arange(rows.shape[1], device=rows.device)
    full, part = lens // p, (lens % p) > 0
    shared = rows[column < full[:, None]].long()
    s["refcount"].index_add_(0, shared, torch.ones_like(shared, dtype=torch.int32))
    fresh = (s["refcount"] == 0).nonzero()[:, 0][: int(part.sum())]
    old = rows[part, full[part].long()].long()
    s["codes"][:, fresh] = s["codes"][:, old]
    s["scales"].view(torch.uint8)[:, fresh] = s["scales"].view(torch.uint8)[:, old]
    rows[part, full[part].long()] = fresh.int()
    s["refcount"][fresh] = 1
    s["block_table"][children] = rows
    s["seq_lens"][children] = lens


def _plain_free(s, seqs):
    rows = s["block_table"][seqs.long()]
    gone = rows[rows >= 0].long()
    s["refcount"].index_add_(0, gone, torch.full_like(gone, -1, dtype=torch.int32))
    s["block_table"][seqs.long()] = -1
    s["seq_lens"][seqs.long()] = 0


def _plain_compact(s):
    live = s["refcount"] > 0
    n = int(live.sum())
    holes, high = (~live[:n]).nonzero()[:, 0], live[n:].nonzero()[:, 0] + n
    s["codes"][:, holes] = s["codes"][:, high]
    s["scales"].view(torch.uint8)[:, holes] = s["scales"].view(torch.uint8)[:, high]
    s["refcount"][holes] = s["refcount"][high]
    s["refcount"][high] = 0
    to = torch.arange(live.numel(), dtype=torch.int32, device=live.device)
    to[high] = holes.int()
    s["block_table"].copy_(torch.where(s["block_table"] >= 0, to[s["block_table"].clamp(min=0).long()], -1))


def _plain_extend(s, seqs, more):
    """Pages for `more` new tokens of each of `seqs`, lowest free ones first; the new tokens' slots."""
    p, at = s["page"], seqs.long()
    old = s["seq_lens"][at]
    have, need = (old + p - 1) // p, (old + more + p - 1) // p
    grow = (need - have).long()
    fresh = (s["refcount"] == 0).nonzero()[:, 0][: int(grow.sum())]
    which = torch.repeat_interleave(torch.arange(at.numel(), device=at.device), grow)
    nth = torch.arange(which.numel(), device=at.device) - (grow.cumsum(0) - grow)[which]
    s["block_table"][at[which], have[which].long() + nth] = fresh.int()
    s["refcount"][fresh] = 1
    s["seq_lens"][at] = old + more
    which = torch.repeat_interleave(torch.arange(at.numel(), device=at.device), more.long())
    pos = torch.arange(which.numel(), device=at.device) - (more.cumsum(0) - more)[which] + old[which]
    return s["block_table"][at[which], pos // p].long() * p + pos % p


def run(s):
    if own:
        return _own(s)
    if s["op"] == "write":
        return _plain_write(s)
    if s["op"] == "attend":
        return _plain_attend(s)
    if s["kind"] == "fork":
        _plain_fork(s)
        out = s["block_table"].clone(), s["refcount"].clone(), s["seq_lens"].clone()
        _plain_free(s, s["children"])
        return out + (s["codes"], s["scales"].view(torch.uint8))
    _plain_free(s, s["drop"])
    _plain_compact(s)
    slots = _plain_extend(s, s["drop"], s["back"])
    return slots, s["block_table"], s["refcount"], s["seq_lens"], s["codes"], s["scales"].view(torch.uint8)


def _own(s):
    if s["op"] == "write":
        from test_speed_scalesweep_b200 import kv_cache
        q = kv_cache.rotary_scalesweep_mse_nvfp4_kv_write(s["q"], s["k"], s["v"], s["positions"], s["table"], s["slots"], s["mult"], s["codes"], s["scales"],
                                                          is_neox=s["neox"])
        k, v = kv_cache.nvfp4_kv_gather(s["codes"], s["scales"], s["mult"], s["slots"], s["q"].dtype)
        return {"query": q, "key": k, "value": v}
    if s["op"] == "attend":
        from test_speed_scalesweep_b200 import kv_attention
        return kv_attention.nvfp4_paged_attention(s["q"], s["codes"], s["scales"], s["mult"], s["block_table"], s["seq_lens"], s["start"], s["max_q"], s["max_s"],
                                                  window=s["window"] or None)
    from test_speed_scalesweep_b200 import kv_pages
    pool = kv_pages.NVFP4KVPages(s["codes"], s["scales"], s["block_table"], s["seq_lens"], s["refcount"])
    if s["kind"] == "fork":
        pool.fork(s["parents"], s["children"])
        out = s["block_table"].clone(), s["refcount"].clone(), s["seq_lens"].clone()
        pool.free(s["children"])
        return out + (s["codes"], s["scales"].view(torch.uint8))
    pool.free(s["drop"])
    pool.compact()
    slots = pool.extend(s["drop"], s["back"], s["total"])
    return slots, s["block_table"], s["refcount"], s["seq_lens"], s["codes"], s["scales"].view(torch.uint8)


# ---- from the definitions, in 64 bits -----------------------------------------------------------------------------
def _exact_block_values(x, mult):
    """What the scale sweep makes of blocks of 16: for each the candidate with the smallest squared error."""
    levels = torch.tensor(E2M1, dtype=torch.float64, device=x.device)
    e4m3 = torch.arange(1, 127, dtype=torch.uint8, device=x.device).view(torch.float8_e4m3fn).double()
    b = (x.double() * mult.double()).reshape(-1, 16)
    target = b.abs().amax(1) / 6
    # the nearest scale; between two, the one with the even code; an all-zero block stays below the first
    near = (target[:, None] - e4m3).abs().argmin(1) + 1
    lower, upper = e4m3[near - 1], e4m3[near.clamp(max=125)]
    near = torch.where((target - lower == upper - target) & (near % 2 == 1), near + 1, near)
    near = torch.where(target <= e4m3[0] / 2, 0, near)
    best, chosen = torch.full_like(target, math.inf), torch.zeros_like(b)
    for step in range(LOWER, LOWER + WINDOW):
        s = e4m3[(near + step).clamp(1, 126) - 1][:, None]
        y = b.abs() / s
        up = torch.bucketize(y, levels).clamp(1, 7)
        a, c = levels[up - 1], levels[up]
        higher = (y - a > c - y) | ((y - a == c - y) & (up % 2 == 0))
        z = torch.where(higher, c, a) * s
        err = (z - b.abs()).square().sum(1)
        wins = err < best
        best = torch.where(wins, err, best)
        chosen = torch.where(wins[:, None], torch.copysign(z, b), chosen)
    return (chosen / mult.double()).view(x.shape)


def exact(case, seed):
    if case["op"] == "pages":
        return None  # whole numbers and copied bytes only
    s = prepare(case, seed)
    if case["op"] == "write":
        half = s["rot"] // 2
        t = s["table"].double()[s["positions"]]
        cis = torch.complex(t[:, :half], t[:, half:])[:, None]

        def turn(x):
            x = x.double()
            head, tail = x[..., : s["rot"]], x[..., s["rot"]:]
            pair = head.unflatten(-1, (2, half)).transpose(-1, -2) if s["neox"] else head.unflatten(-1, (half, 2))
            z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * cis)
            z = (z.transpose(-1, -2) if s["neox"] else z).flatten(-2)
            return torch.cat([z, tail], -1)

        skip = (s["slots"] < 0)[:, None, None]
        # a key is rounded to its type before it is quantized
        key = _exact_block_values(turn(s["k"]).to(s["k"].dtype), s["mult"][0])
        value = _exact_block_values(s["v"].contiguous(), s["mult"][1])
        return {"query": turn(s["q"]), "key": key.masked_fill(skip, 0.0), "value": value.masked_fill(skip, 0.0)}
    seq, qry = _lengths(case)
    signed = torch.tensor(E2M1 + tuple(-e for e in E2M1), dtype=torch.float64, device="cuda")
    out, at = [], 0
    for i, (n, m) in enumerate(zip(seq, qry)):
        ids = s["block_table"][i, : -(-n // s["page"])].long()
        heads = []
        for h in range(s["hkv"]):
            dense = []
            for side in (0, 1):
                c = s["codes"][ids, side, h].reshape(-1, s["d"] // 2)[:n]
                w = s["scales"].view(torch.uint8)[ids, side, h].reshape(-1, s["d"] // 16)[:n].contiguous().view(torch.float8_e4m3fn).double()
                x = signed[torch.stack([c % 16, c // 16], -1).long()].reshape(n, -1, 16) * w[:, :, None] / s["mult"][side].double()
                dense.append(x.reshape(n, -1))
            g = s["hq"] // s["hkv"]
            query = s["q"][at:at + m, h * g:(h + 1) * g].double().transpose(0, 1)
            for one in query.split(1):  # one query head at a time: the scores of a long prompt are large
                logit = one[0] @ dense[0].T / math.sqrt(s["d"])
                sees = torch.arange(n, device="cuda")[None] - torch.arange(n - m, n, device="cuda")[:, None]
                keep = (sees <= 0) & ((sees >= -s["window"]) if s["window"] else True)
                heads.append(torch.softmax(logit.masked_fill(~keep, -math.inf), -1) @ dense[1])
        out.append(torch.stack(heads, 1))
        at += m
    return torch.cat(out)
