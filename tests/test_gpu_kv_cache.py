"""GPU parity of the rotary + scale-sweep cache write and of the gather: the
cache's bytes against the CPU oracle's quantizer on keys rotated in binary32,
the query bit for bit, both directions of the format, and what the write must
leave alone."""
import numpy as np
import pytest
import torch

import oracle

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16}
MULT = (1536.0 / 23.17, 1536.0 / 21.91)
SENTINEL = 0xA5


@pytest.fixture(scope="module")
def kv(built_library):
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from test_speed_scalesweep_b200 import kv_cache
    return kv_cache


def rotate(x, table, pos, neox):
    """Rotary positions in binary32 on the CPU: torch rounds every product and sum."""
    rot = table.shape[1]
    row = table[pos][:, None]
    c, s = row[..., : rot // 2], row[..., rot // 2:]
    y = x.float()
    a, b = (y[..., : rot // 2], y[..., rot // 2: rot]) if neox else (y[..., 0:rot:2], y[..., 1:rot:2])
    oa, ob = a * c - b * s, b * c + a * s
    turned = torch.cat([oa, ob], -1) if neox else torch.stack([oa, ob], -1).flatten(-2)
    return torch.cat([turned, y[..., rot:]], -1).to(x.dtype)


def bits(t):
    return t.contiguous().view(torch.int16).numpy().view(np.uint16)


def expect(x, mult, dtype):
    """Codes [T, H, D/2] and scales [T, H, D/16] of the oracle's quantizer."""
    t, h, d = x.shape
    codes, scales = oracle.quantize(bits(x).reshape(t * h, d), float(np.float32(mult)), dtype=dtype,
                                    swizzled=False)
    return codes.reshape(t, h, d // 2), scales.reshape(t, h, d // 16)


def make(t, hq, hkv, d, dtype, page, seed, specials=False, layers=None):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(t, hq + 2 * hkv, d, generator=g) * torch.exp(
        0.7 * torch.randn(hq + 2 * hkv, d, generator=g))
    if specials and t:
        flat = qkv.view(-1)
        at = torch.randperm(flat.numel(), generator=g)[:40]
        for i, v in enumerate((float("inf"), float("-inf"), float("nan"), -0.0, 1e-30, 1e4, 0.0, -1e4)):
            flat[at[i::8]] = v
        qkv[0, -1] = 0.0
    qkv = qkv.to(DT[dtype])
    pages = -(-t // page) + 2
    slots = torch.randperm(pages * page, generator=g)[:t]
    pos = torch.randint(0, 5000, (t,), generator=g)
    return qkv, slots, pos, pages


def check(kv, t, hq, hkv, d, rot, neox, dtype, page, seed=0, specials=False, in_place=False):
    qkv, slots, pos, pages = make(t, hq, hkv, d, dtype, page, seed, specials)
    table = kv.rotary_cos_sin_cache(5000, rot, device="cpu")
    if t > 4:
        slots[1], slots[3] = -1, pages * page + 5  # padding
    dev = qkv.cuda()
    q, k, v = dev[:, :hq], dev[:, hq:hq + hkv], dev[:, hq + hkv:]
    codes, scales = kv.alloc_kv_cache(pages, page, hkv, d)
    codes.fill_(SENTINEL)
    scales.view(torch.uint8).fill_(SENTINEL)
    mult = torch.tensor(MULT).cuda()
    out = kv.rotary_scalesweep_mse_nvfp4_kv_write(
        q, k, v, pos.cuda(), table.cuda(), slots.cuda(), mult, codes, scales, is_neox=neox,
        query_out=q if in_place else None)
    torch.cuda.synchronize()
    x = qkv
    rq, rk = rotate(x[:, :hq], table, pos, neox), rotate(x[:, hq:hq + hkv], table, pos, neox)
    got, want = out.cpu().contiguous(), rq.contiguous()
    same = (got.view(torch.int16) == want.view(torch.int16)) | (got.isnan() & want.isnan())
    assert bool(same.all()), int((~same).sum())
    # keys and values as they were (the query too, unless it was rotated in place)
    rest = slice(hq, None) if in_place else slice(None)
    assert torch.equal(dev.cpu()[:, rest].contiguous().view(torch.int16), x[:, rest].contiguous().view(torch.int16))
    want_c = np.full(tuple(codes.shape), SENTINEL, np.uint8)
    want_s = np.full(tuple(scales.shape), SENTINEL, np.uint8)
    for side, y in ((0, rk), (1, x[:, hq + hkv:])):
        ec, es = expect(y, MULT[side], dtype)
        for i, slot in enumerate(slots.tolist()):
            if 0 <= slot < pages * page:
                want_c[slot // page, side, :, slot % page] = ec[i]
                want_s[slot // page, side, :, slot % page] = es[i]
    assert np.array_equal(codes.cpu().numpy(), want_c)
    assert np.array_equal(scales.view(torch.uint8).cpu().numpy(), want_s)
    # and back: code * (scale / multiplier), both rounded to binary32, then to the type
    gk, gv = kv.nvfp4_kv_gather(codes, scales, mult, slots.cuda(), DT[dtype])
    for side, g in ((0, gk), (1, gv)):
        live = (slots >= 0) & (slots < pages * page)
        at = slots[live]
        c = want_c[at // page, side, :, at % page].reshape(-1, d // 2)
        s = want_s[at // page, side, :, at % page].reshape(-1, d // 16)
        one = np.full_like(s, 0x38)  # an E4M3 scale of 1
        code = oracle.dequantize(c, one, c.shape[0], d, swizzled=False)
        factor = (torch.from_numpy(s).view(torch.float8_e4m3fn).float().numpy() / np.float32(MULT[side]))
        val = code * factor.repeat(16, axis=1)
        assert val.dtype == np.float32
        full = torch.zeros(t, hkv, d, dtype=DT[dtype])
        full[live] = torch.from_numpy(val).reshape(-1, hkv, d).to(DT[dtype])
        assert torch.equal(g.cpu().float(), full.float())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("t,hq,hkv,d,rot,page", [
    (1, 32, 8, 128, 128, 16), (7, 5, 1, 64, 16, 16), (33, 6, 3, 256, 80, 32),
    (129, 4, 2, 128, 48, 128), (1000, 8, 2, 64, 64, 64), (257, 16, 16, 256, 256, 16)])
def test_bytes_match_the_oracle(kv, t, hq, hkv, d, rot, page, neox, dtype):
    check(kv, t, hq, hkv, d, rot, neox, dtype, page, seed=t)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_special_values_and_in_place_query(kv, dtype):
    check(kv, 65, 4, 2, 128, 64, True, dtype, 16, seed=3, specials=True, in_place=True)
    check(kv, 65, 4, 2, 128, 64, False, dtype, 16, seed=4, specials=True, in_place=True)


def test_no_tokens_and_positions_outside_the_table(kv):
    codes, scales = kv.alloc_kv_cache(2, 16, 1, 64)
    codes.fill_(SENTINEL)
    mult, table = torch.tensor(MULT).cuda(), kv.rotary_cos_sin_cache(10, 64)
    x = torch.randn(3, 1, 64, device="cuda").bfloat16()
    empty = torch.empty(0, dtype=torch.int64, device="cuda")
    out = kv.rotary_scalesweep_mse_nvfp4_kv_write(x[:0], x[:0], x[:0], empty, table, empty, mult,
                                                  codes, scales)
    assert out.shape == (0, 1, 64)
    assert kv.nvfp4_kv_gather(codes, scales, mult, empty)[0].shape == (0, 1, 64)
    pos = torch.tensor([9, 10, -1], device="cuda")
    out = kv.rotary_scalesweep_mse_nvfp4_kv_write(x, x, x, pos, table,
                                                  torch.arange(3, device="cuda"), mult, codes, scales)
    assert bool(out[0].isfinite().all()) and bool(out[1:].isnan().all())
    assert bool((codes[0, :, :, 1:] == SENTINEL).all()) and bool((codes[0, :, :, 0] != SENTINEL).any())


def test_layer_of_a_cache_other_stream_and_graph(kv):
    qkv, slots, pos, pages = make(40, 4, 2, 64, "bf16", 16, seed=9)
    dev, table, mult = qkv.cuda(), kv.rotary_cos_sin_cache(5000, 64), torch.tensor(MULT).cuda()
    codes, scales = kv.alloc_kv_cache(pages, 16, 2, 64, num_layers=3)
    codes.fill_(SENTINEL)
    scales.view(torch.uint8).fill_(SENTINEL)
    one = [t.clone() for t in (codes[0], scales[0])]
    args = (dev[:, :4], dev[:, 4:6], dev[:, 6:], pos.cuda(), table, slots.cuda(), mult)
    want = kv.rotary_scalesweep_mse_nvfp4_kv_write(*args, *one)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        got = kv.rotary_scalesweep_mse_nvfp4_kv_write(*args, codes[1], scales[1])
    stream.synchronize()
    assert torch.equal(got, want) and torch.equal(codes[1], one[0])
    assert torch.equal(scales[1].view(torch.uint8), one[1].view(torch.uint8))
    assert bool((codes[0] == SENTINEL).all()) and bool((codes[2] == SENTINEL).all())
    # captured, replayed on new values
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kv.rotary_scalesweep_mse_nvfp4_kv_write(*args, codes[2], scales[2])
    dev.copy_(dev.flip(0))
    graph.replay()
    want = kv.rotary_scalesweep_mse_nvfp4_kv_write(*args, *one)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(codes[2], one[0])


def test_refusals_of_tensors(kv):
    """Everything that Python can pass wrongly is an error before a kernel runs."""
    from test_speed_scalesweep_b200 import kv_attention
    codes, scales = kv.alloc_kv_cache(4, 16, 2, 64)
    mult, table = torch.ones(2, device="cuda"), kv.rotary_cos_sin_cache(8, 64)
    x = torch.zeros(3, 2, 64, device="cuda", dtype=torch.bfloat16)
    idx = torch.zeros(3, dtype=torch.int64, device="cuda")

    def write(query=x, key=x, value=x, positions=idx, cos_sin=table, slots=idx, scale=mult, c=codes, s=scales, **kw):
        return kv.rotary_scalesweep_mse_nvfp4_kv_write(query, key, value, positions, cos_sin, slots, scale, c, s, **kw)

    wide = torch.zeros(3, 2, 68, device="cuda", dtype=torch.bfloat16)[..., :64]
    for match, kw in (
            ("shape", dict(key=x[:2])), ("shape", dict(value=x[:, :1])), ("shape", dict(key=x.half())),
            ("head size", dict(query=x[..., :32])), ("T, heads", dict(query=x[0])), ("bfloat16", dict(query=x.float())),
            ("multiples of 8", dict(key=wide)), ("contiguous", dict(value=x.transpose(1, 2).contiguous().transpose(1, 2))),
            ("on cuda", dict(key=x.cpu())), ("int64", dict(positions=idx.int())), ("int64", dict(slots=idx[:2])),
            ("int64", dict(slots=idx.cpu())), ("cos_sin_cache", dict(cos_sin=table.double())),
            ("cos_sin_cache", dict(cos_sin=table.t())), ("rotary_dim", dict(cos_sin=table[:, :24].contiguous())),
            ("kv_input_scale", dict(scale=mult[:1])), ("kv_input_scale", dict(scale=None)),
            ("within a page", dict(c=torch.zeros(4, 2, 16, 2, 32, dtype=torch.uint8, device="cuda").transpose(2, 3))),
            ("expanded", dict(query_out=x[:1].expand(3, 2, 64))), ("query_out", dict(query_out=x[:2])),
            ("16-byte", dict(query=torch.zeros(3 * 128 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(3, 2, 64)))):
        with pytest.raises(ValueError, match=match):
            write(**kw)
    tab, lens, start = (torch.zeros(s, dtype=torch.int32, device="cuda") for s in ((2, 4), (2,), (3,)))

    def attend(q=x, t=tab, n=lens, s=start, mq=1, ms=16, **kw):
        return kv_attention.nvfp4_paged_attention(q, codes, scales, mult, t, n, s, mq, ms, **kw)

    for match, kw in (
            ("multiple of the cache", dict(q=x[:, :1])), ("block_table", dict(t=tab.long())), ("block_table", dict(t=tab[0])),
            ("contiguous", dict(t=tab.t().contiguous().t())), ("seq_lens", dict(n=lens[:1])), ("query_start", dict(s=start[:2])),
            ("query_start", dict(s=start.cpu())), ("max_query_len", dict(mq=0)), ("max_query_len", dict(ms=0)),
            ("integer", dict(mq=1.5)), ("window", dict(window=-1)), ("finite", dict(softmax_scale=float("nan"))),
            ("number", dict(softmax_scale="x")), ("status", dict(status=lens.long())), ("out", dict(out=x.half())),
            ("expanded", dict(out=x[:1].expand(3, 2, 64)))):
        with pytest.raises(ValueError, match=match):
            attend(**kw)
    before = codes.clone()
    assert write(query=x[:0], key=x[:0], value=x[:0], positions=idx[:0], slots=idx[:0]).shape == (0, 2, 64)
    assert attend(q=x[:0]).shape == (0, 2, 64)
    assert torch.equal(codes, before)
