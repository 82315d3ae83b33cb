"""GPU checks of the workspace that attention asks for: no more than the rows
that are split need, all of it written before it is read, nothing behind it."""
import ctypes

import pytest
import torch

from test_gpu_kv_attention import Batch, attn  # noqa: F401  (attn: the fixture)

pytestmark = pytest.mark.gpu

MIB = 1 << 20


def arguments(hq, hkv, d, seqs, tokens, max_q, max_s, page=16):
    """(cache, attention) structs whose sizes alone matter."""
    from test_speed_scalesweep_b200 import _lib
    cache = _lib.KVCache(codes=1 << 20, scales=1 << 20, codes_page_stride=hkv * page * d,
                         scales_page_stride=hkv * page * d // 8, input_scale=1 << 20, num_pages=4, page_size=page,
                         kv_heads=hkv, head_size=d)
    args = _lib.KVAttention(block_table=1 << 20, block_table_stride=8, seq_lens=1 << 20, query_start=1 << 20,
                            tokens=tokens, seqs=seqs, block_table_columns=8, q_heads=hq, max_query_len=max_q,
                            max_seq_len=max_s, causal=1, window=-1, softmax_scale=0.1)
    return cache, args


def need(*a, **kw):
    from test_speed_scalesweep_b200 import _lib
    cache, args = arguments(*a, **kw)
    n = _lib.lib().ssw_nvfp4_paged_attention_workspace_bytes(ctypes.byref(cache), ctypes.byref(args), 0)
    assert n >= 0
    return n


@pytest.mark.parametrize("hq,hkv,d,prompt,singles,keys", [
    (32, 8, 128, 8192, 1, 131072), (32, 8, 128, 8192, 1, 32768), (64, 8, 128, 8192, 8, 131072),
    (32, 8, 128, 8191, 3, 131072), (16, 1, 256, 4096, 2, 1 << 20), (24, 6, 64, 333, 23, 3001)])
def test_prompts_beside_single_tokens(attn, hq, hkv, d, prompt, singles, keys):  # noqa: F811
    """What is split is at most 8 or 16 rows of a sequence and kv head, in at most 24 parts for each of 148
    multiprocessors and one a sequence and head more, or, of the prompts, four waves of tiles of 256 rows."""
    rows = 8 if hq // hkv <= 8 else 16
    parts = 24 * 148 + 2 * (singles + 1) * hkv
    most = max(parts * rows, 4 * 148 * 256 + hq * (prompt + singles) * (singles + 2)) * (d + 2) * 4
    got = need(hq, hkv, d, 1 + singles, prompt + singles, prompt, keys)
    assert got <= min(most, 128 * MIB), (got, most)


@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (24, 6, 64), (8, 1, 256), (32, 2, 128)])
@pytest.mark.parametrize("seqs,keys", [(2, 131072), (5, 30000), (24, 8192)])
def test_single_tokens_beside_prompts_are_cut_as_alone(attn, hq, hkv, d, seqs, keys):  # noqa: F811
    tile = 8 if hq // hkv <= 8 else 16
    prompt = 128  # one tile or two of each sequence, whose own partial results are smaller
    mixed, alone = need(hq, hkv, d, seqs, seqs * prompt, prompt, keys), need(hq, hkv, d, seqs, seqs, 1, keys)
    splits, rest = divmod(alone, seqs * hq * (d + 2) * 4)
    assert rest == 0 and splits > 1
    assert mixed >= splits * seqs * hkv * tile * (d + 2) * 4


@pytest.mark.parametrize("hq,hkv,d,seqs,max_q", [(32, 8, 128, 1, 1), (8, 8, 64, 3, 2), (16, 2, 128, 2, 100)])
def test_a_padded_query_tensor_costs_nothing(attn, hq, hkv, d, seqs, max_q):  # noqa: F811
    tight = need(hq, hkv, d, seqs, seqs * max_q, max_q, 65536)
    assert 0 < tight <= need(hq, hkv, d, seqs, 1 << 16, max_q, 65536)
    # rows kept per sequence are rounded up to whole tiles of 8, 16 or 256 rows
    group = hq // hkv
    tile = 8 if max_q * group <= 8 else 16 if max_q * group <= 32 else 256
    whole = -(-max_q * group // tile) * tile
    assert need(hq, hkv, d, seqs, 1 << 16, max_q, 65536) <= tight * whole / (max_q * group)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("lens,hq,hkv,d,pad", [
    ([(40, 30), (9000, 1), (7000, 2), (3, 3), (5000, 40)], 8, 2, 128, 0), ([(200, 150), (30000, 1)], 8, 2, 64, 0),
    ([(5000, 1)], 8, 2, 128, 300), ([(4000, 3), (3000, 1)], 20, 2, 128, 500), ([(6000, 2)], 4, 1, 256, 100),
    ([(3000, 100), (2500, 70)], 4, 2, 128, 900), ([(3000, 60), (20, 1), (9000, 1)], 16, 1, 256, 0)])
def test_written_before_it_is_read_and_nothing_behind(attn, lens, hq, hkv, d, pad, dtype):  # noqa: F811
    from test_speed_scalesweep_b200 import _lib
    lib = _lib.lib()
    b = Batch(lens, hq, hkv, d, 16, dtype, seed=31)
    rows = b.q.shape[0]
    q = torch.cat([b.q, torch.full((pad, hq, d), float("nan"), dtype=b.dtype, device="cuda")])
    out = torch.full_like(q, 3.0)
    lse = torch.full((rows + pad, hq), 3.0, device="cuda")
    cache = _lib.KVCache(codes=b.codes.data_ptr(), scales=b.raw.data_ptr(), codes_page_stride=b.codes.stride(0),
                         scales_page_stride=b.raw.stride(0), input_scale=b.mult.data_ptr(),
                         num_pages=b.codes.shape[0], page_size=16, kv_heads=hkv, head_size=d)
    args = _lib.KVAttention(block_table=b.table.data_ptr(), block_table_stride=b.table.stride(0),
                            seq_lens=b.seq_lens.data_ptr(), query_start=b.start.data_ptr(), lse=lse.data_ptr(),
                            tokens=rows + pad, seqs=len(lens), block_table_columns=b.table.shape[1], q_heads=hq,
                            max_query_len=b.max_q, max_seq_len=b.max_s, causal=1, window=-1, softmax_scale=d ** -0.5)
    code = 0 if dtype == "bf16" else 1
    size = lib.ssw_nvfp4_paged_attention_workspace_bytes(ctypes.byref(cache), ctypes.byref(args), code)
    assert size > 0
    ws = torch.full((size // 4 + 4096,), float("nan"), device="cuda")
    heads = [_lib.KVHeads(t.data_ptr(), hq * d, d) for t in (q, out)]
    for _ in range(2):  # the second call finds the first one's partial results
        assert lib.ssw_nvfp4_paged_attention(ctypes.byref(cache), ctypes.byref(args), code, ctypes.byref(heads[0]),
                                             ctypes.byref(heads[1]), ws.data_ptr(), size,
                                             torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        b.check(out[:rows], lse[:rows])
        assert bool((out[rows:] == 3).all()) and bool((lse[rows:] == 3).all())
        assert bool(ws[size // 4:].isnan().all())


def test_memory_of_a_call(attn):  # noqa: F811
    b = Batch([(8192, 8191), (60000, 1)], 32, 8, 128, 16, "bf16", seed=32)
    out = torch.empty_like(b.q)
    b.call(attn, out=out)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    b.call(attn, out=out)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - before <= 128 * MIB
