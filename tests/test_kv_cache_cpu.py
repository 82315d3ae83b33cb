"""Host side of the KV-cache operators: refusals, allocation and the rotary
table, without a GPU."""
import ctypes
import math

import pytest
import torch

from test_speed_scalesweep_b200 import _lib, kv_cache


def cache(**kw):
    d = dict(codes=0x10000, scales=0x20000, codes_page_stride=2 * 2 * 16 * 64,
             scales_page_stride=2 * 2 * 16 * 8, input_scale=0x3000, num_pages=4, page_size=16,
             kv_heads=2, head_size=128)
    d.update(kw)
    return _lib.KVCache(**d)


def heads(data=0x40000, token_stride=1024, head_stride=128):
    return _lib.KVHeads(data, token_stride, head_stride)


def write(c=None, dtype=0, tokens=4, hq=4, q=None, k=None, pos=0x5000, table=0x6000, maxp=8,
          rot=64, slots=0x7000):
    h = heads()
    return _lib.lib().ssw_rotary_scalesweep_mse_nvfp4_kv_write(
        ctypes.byref(c or cache()), dtype, tokens, hq, ctypes.byref(q or h), ctypes.byref(k or h),
        ctypes.byref(h), ctypes.byref(h), pos, table, maxp, rot, 1, slots, None)


@pytest.mark.parametrize("kw,needle", [
    (dict(c=dict(head_size=96)), "head_size"), (dict(c=dict(page_size=24)), "page_size"),
    (dict(c=dict(kv_heads=0)), "kv_heads"), (dict(c=dict(codes_page_stride=1024)), "overlap"),
    (dict(c=dict(codes_page_stride=4104)), "multiples of 16"), (dict(c=dict(codes=0x10008)), "16-byte"),
    (dict(c=dict(scales=0)), "null"), (dict(c=dict(input_scale=0)), "null"),
    (dict(dtype=2), "dtype"), (dict(tokens=-1), "bad sizes"), (dict(tokens=1 << 40), "too many"),
    (dict(rot=24), "rotary_dim"), (dict(rot=144), "rotary_dim"), (dict(rot=0), "rotary_dim"),
    (dict(maxp=0), "empty"), (dict(q=heads(data=0)), "null query"),
    (dict(k=heads(token_stride=1028)), "key"), (dict(q=heads(data=0x40008)), "query"),
    (dict(pos=None), "null"), (dict(slots=None), "null"), (dict(table=0x6004), "misaligned")])
def test_write_refusals(built_library, kw, needle):
    kw = dict(kw)
    if "c" in kw:
        kw["c"] = cache(**kw["c"])
    st = write(**kw)
    assert st == _lib.SSW_ERR_INVALID_ARGUMENT
    with pytest.raises(ValueError, match=needle):
        _lib.check(st)


def test_no_tokens_is_a_no_op(built_library):
    assert write(tokens=0, pos=None, slots=None) == 0
    assert _lib.lib().ssw_nvfp4_kv_gather(ctypes.byref(cache()), 0, 0, None, None, None, None) == 0


def test_python_refuses_cpu_and_wrong_tensors(built_library):
    codes, scales = kv_cache.alloc_kv_cache(2, 16, 1, 64, device="cpu")
    assert codes.shape == (2, 2, 1, 16, 32) and scales.shape == (2, 2, 1, 16, 4)
    mult, slots = torch.ones(2), torch.zeros(1, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        kv_cache.nvfp4_kv_gather(codes, scales, mult, slots)
    with pytest.raises(ValueError, match="head_size/16"):
        kv_cache.nvfp4_kv_gather(codes, scales[..., :2], mult, slots)
    with pytest.raises(ValueError, match="uint8"):
        kv_cache.nvfp4_kv_gather(codes.int(), scales, mult, slots)
    with pytest.raises(ValueError, match="num_pages"):
        kv_cache.nvfp4_kv_gather(codes[0], scales[0], mult, slots)
    with pytest.raises(ValueError, match="codes must be a tensor"):
        kv_cache.nvfp4_kv_gather(None, scales, mult, slots)
    with pytest.raises(ValueError, match="bfloat16"):
        kv_cache.nvfp4_kv_gather(codes, scales, mult, slots, torch.float32)
    for bad in (dict(page_size=24), dict(head_size=80), dict(num_pages=0), dict(num_layers=0)):
        with pytest.raises(ValueError):
            kv_cache.alloc_kv_cache(**{**dict(num_pages=2, page_size=16, kv_heads=1, head_size=64,
                                              device="cpu"), **bad})


def test_rotary_table():
    t = kv_cache.rotary_cos_sin_cache(200001, 8, base=500000.0, device="cpu")
    assert t.shape == (200001, 8) and t.dtype == torch.float32
    angle = 200000 * 500000.0 ** (-2 / 8)
    # a binary64 angle near 2e5 is off by 2^-36 at most, the float32 result by half a step of a value up to 1
    assert abs(t[200000, 1].item() - math.cos(angle)) < 2 ** -24
    assert abs(t[200000, 5].item() - math.sin(angle)) < 2 ** -24
    lin = kv_cache.rotary_cos_sin_cache(9, 8, scaling={"rope_type": "linear", "factor": 4}, device="cpu")
    assert torch.equal(lin[8], kv_cache.rotary_cos_sin_cache(9, 8, device="cpu")[2])
    with pytest.raises(ValueError, match="rope_type"):
        kv_cache.rotary_cos_sin_cache(9, 8, scaling={"rope_type": "spiral"}, device="cpu")
    with pytest.raises(ValueError, match="even"):
        kv_cache.rotary_cos_sin_cache(9, 7, device="cpu")
    for extra in ({"mscale": 1.0}, {"mscale_all_dim": 0.7}, {"truncate": False}):
        with pytest.raises(ValueError, match="attention_factor"):
            kv_cache.rotary_cos_sin_cache(9, 8, device="cpu", scaling=dict(
                extra, rope_type="yarn", factor=4.0, original_max_position_embeddings=64))


@pytest.mark.parametrize("scaling", [
    {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
     "original_max_position_embeddings": 8192},
    {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}])
def test_scaled_frequencies_match_transformers(scaling):
    rope = pytest.importorskip("transformers.modeling_rope_utils")

    class Config:
        rope_theta, head_dim, hidden_size, num_attention_heads = 500000.0, 128, 4096, 32
        max_position_embeddings, partial_rotary_factor = 131072, 1.0
        rope_scaling = dict(scaling)
        rope_parameters = dict(scaling, rope_theta=500000.0)

        def standardize_rope_params(self):
            return None
    inv, factor = rope.ROPE_INIT_FUNCTIONS[scaling["rope_type"]](Config(), torch.device("cpu"))
    got = kv_cache.rotary_cos_sin_cache(2, 128, 500000.0, scaling, device="cpu")[1]
    # its frequencies are float32 from a handful of float32 steps: 8 half steps of 2^-24, on an
    # angle of at most 1 whose sine and cosine move no faster
    tol = 8 * 2 ** -24 + 2 ** -24
    assert torch.allclose(got[:64], inv.cos() * factor, rtol=0, atol=tol * factor)
    assert torch.allclose(got[64:], inv.sin() * factor, rtol=0, atol=tol * factor)


def attention(dtype=0, c=None, **kw):
    d = dict(block_table=0x1000, block_table_stride=4, seq_lens=0x2000, query_start=0x3000, tokens=4,
             seqs=2, block_table_columns=4, q_heads=4, max_query_len=2, max_seq_len=64, causal=1,
             window=-1, softmax_scale=0.1)
    d.update(kw)
    h = heads()
    return _lib.lib().ssw_nvfp4_paged_attention(ctypes.byref(c or cache()), ctypes.byref(_lib.KVAttention(**d)),
                                                dtype, ctypes.byref(h), ctypes.byref(h), None, 0, None)


@pytest.mark.parametrize("kw,needle", [
    (dict(q_heads=3), "multiple of the cache"), (dict(q_heads=0), "multiple of the cache"),
    (dict(tokens=-1), "bad sizes"), (dict(tokens=1 << 40), "bad sizes"), (dict(seqs=-1), "bad sizes"),
    (dict(max_query_len=0), "max_query_len"), (dict(max_seq_len=0), "max_query_len"),
    (dict(max_seq_len=(1 << 30) + 1), "max_query_len"), (dict(max_query_len=1 << 30), "max_query_len"),
    (dict(seqs=1 << 30, max_query_len=1 << 20), "too many"), (dict(block_table_columns=0), "block table"), (dict(block_table_stride=3), "block table"),
    (dict(softmax_scale=math.inf), "finite"), (dict(softmax_scale=math.nan), "finite"),
    (dict(block_table=None), "null"), (dict(seq_lens=None), "null"), (dict(query_start=0x3002), "misaligned"),
    (dict(dtype=5), "dtype"), (dict(c=cache(head_size=192)), "head_size")])
def test_attention_refusals(built_library, kw, needle):
    st = attention(**kw)
    assert st == _lib.SSW_ERR_INVALID_ARGUMENT
    with pytest.raises(ValueError, match=needle):
        _lib.check(st)


def test_attention_of_nothing_is_a_no_op(built_library):
    assert attention(tokens=0) == 0 and attention(seqs=0) == 0


def tables(**kw):
    d = dict(refcount=0x1000, block_table=0x2000, table_stride=4, seq_lens=0x3000, status=None,
             num_pages=8, max_seqs=4, columns=4, page_size=16)
    d.update(kw)
    return _lib.KVPages(**d)


def pool(**kw):
    d = dict(codes=0x10000, scales=0x20000, codes_layer_stride=1 << 16, scales_layer_stride=1 << 13,
             codes_page_stride=4096, scales_page_stride=512, codes_page_bytes=4096, scales_page_bytes=512,
             num_pages=8, layers=2)
    d.update(kw)
    return _lib.KVPool(**d)


WS = (0x40000, 1 << 20, None)


@pytest.mark.parametrize("call,needle", [
    (lambda h: h.ssw_kv_pages_free(ctypes.byref(tables(page_size=8)), 1, 0x100, None), "page_size"),
    (lambda h: h.ssw_kv_pages_free(ctypes.byref(tables(table_stride=3)), 1, 0x100, None), "bad sizes"),
    (lambda h: h.ssw_kv_pages_free(ctypes.byref(tables()), 5, 0x100, None), "has 4"),
    (lambda h: h.ssw_kv_pages_free(ctypes.byref(tables()), 1, None, None), "null"),
    (lambda h: h.ssw_kv_pages_free(ctypes.byref(tables(refcount=None)), 1, 0x100, None), "null"),
    (lambda h: h.ssw_kv_pages_free(ctypes.byref(tables()), 1, 0x102, None), "misaligned"),
    (lambda h: h.ssw_kv_pages_fork(ctypes.byref(tables()), ctypes.byref(pool(num_pages=9)), 1, 0x100, 0x200, *WS), "the tables 8"),
    (lambda h: h.ssw_kv_pages_fork(ctypes.byref(tables()), ctypes.byref(pool(codes_page_bytes=24)), 1, 0x100, 0x200, *WS), "multiple of 16"),
    (lambda h: h.ssw_kv_pages_fork(ctypes.byref(tables()), ctypes.byref(pool(scales_page_stride=496)), 1, 0x100, 0x200, *WS), "overlap"),
    (lambda h: h.ssw_kv_pages_fork(ctypes.byref(tables()), ctypes.byref(pool(layers=0)), 1, 0x100, 0x200, *WS), "layers"),
    (lambda h: h.ssw_kv_pages_fork(ctypes.byref(tables()), ctypes.byref(pool()), 1, 0x100, 0x200, 0x40000, 8, None), "workspace"),
    (lambda h: h.ssw_kv_pages_extend(ctypes.byref(tables()), 1, 0x100, 0x200, -1, 0x300, *WS), "new tokens"),
    (lambda h: h.ssw_kv_pages_extend(ctypes.byref(tables()), 0, None, None, 1, 0x300, *WS), "new tokens"),
    (lambda h: h.ssw_kv_pages_extend(ctypes.byref(tables()), 1, 0x100, 0x200, 1, None, *WS), "slot_mapping"),
    (lambda h: h.ssw_kv_pages_extend(ctypes.byref(tables()), 1, 0x100, 0x200, 1, 0x300, None, 0, None), "workspace"),
    (lambda h: h.ssw_kv_pages_compact(ctypes.byref(tables()), ctypes.byref(pool()), 0x40002, 1 << 20, None), "workspace"),
    (lambda h: h.ssw_kv_pages_compact(ctypes.byref(tables()), ctypes.byref(pool(codes=None)), *WS), "null"),
    (lambda h: h.ssw_kv_pages_copy(ctypes.byref(pool()), -1, 0x100, 0x200, None), "bad size"),
    (lambda h: h.ssw_kv_pages_copy(ctypes.byref(pool()), 1, 0x100, None, None), "null")])
def test_pages_refusals(built_library, call, needle):
    st = call(_lib.lib())
    assert st == _lib.SSW_ERR_INVALID_ARGUMENT
    with pytest.raises(ValueError, match=needle):
        _lib.check(st)


def test_pages_python_refusals(built_library):
    from test_speed_scalesweep_b200 import kv_pages
    codes, scales = kv_cache.alloc_kv_cache(4, 16, 1, 64, device="cpu", num_layers=2)
    with pytest.raises(ValueError, match="CUDA"):
        kv_pages.NVFP4KVPages.empty(codes, scales, 2, 2)
    with pytest.raises(ValueError, match="num_pages"):
        kv_pages.NVFP4KVPages.empty(codes[0, 0], scales[0, 0], 2, 2)
    with pytest.raises(ValueError, match="head_size/16"):
        kv_pages.NVFP4KVPages.empty(codes, scales[..., :2], 2, 2)


def test_ops_registered_with_fake_shapes():
    from test_speed_scalesweep_b200 import ops  # noqa: F401
    ns = torch.ops.scalesweep_b200
    codes, scales = kv_cache.alloc_kv_cache(8, 16, 2, 128, device="meta")
    q = torch.empty(5, 4, 128, dtype=torch.bfloat16, device="meta")
    kv = torch.empty(5, 2, 128, dtype=torch.bfloat16, device="meta")
    idx, mult = torch.empty(5, dtype=torch.int64, device="meta"), torch.empty(2, device="meta")
    table = torch.empty(64, 128, device="meta")
    out = ns.rotary_scalesweep_mse_nvfp4_kv_write(q, kv, kv, idx, table, idx, mult, codes, scales, True)
    assert out.shape == q.shape and out.dtype == q.dtype
    i32 = [torch.empty(s, dtype=torch.int32, device="meta") for s in ((1, 4), (1,), (2,))]
    assert ns.nvfp4_paged_attention(q, codes, scales, mult, *i32, 5, 64).shape == q.shape
    k, v = ns.nvfp4_kv_gather(codes, scales, mult, idx, torch.float16)
    assert k.shape == v.shape == (5, 2, 128) and k.dtype == torch.float16
