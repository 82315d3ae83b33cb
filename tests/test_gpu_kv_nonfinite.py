"""GPU checks of attention over the NVFP4 cache where queries hold NaN or
infinities: such a row is NaN as the formula has it, however the call is cut,
and no other row notices."""
import pytest
import torch

from test_gpu_kv_attention import Batch, attn  # noqa: F401  (attn: the fixture)

pytestmark = pytest.mark.gpu

CUTS = {  # (lengths, hq, hkv, d, page)
    "one tile, one split": ([(100, 1), (7, 1), (0, 1)], 4, 1, 128, 16),
    "few splits": ([(700, 1)], 4, 1, 128, 16),
    "many splits": ([(5000, 1)], 8, 2, 128, 32),
    "16 rows": ([(900, 3), (40, 2)], 10, 2, 128, 16),
    "32 rows": ([(600, 8), (3, 7)], 4, 1, 64, 64),
    "two tiles": ([(600, 8), (3, 7)], 4, 1, 128, 64),
    "heads of 256": ([(90, 2), (1, 2)], 4, 1, 256, 16),
    "heads of 256, splits": ([(900, 2), (1, 2)], 4, 1, 256, 16),
    "prompt": ([(200, 150), (129, 65), (3, 7)], 8, 8, 64, 16),
    "prompt of several tiles": ([(600, 600)], 8, 2, 128, 16),
    "prompt, splits": ([(2000, 150)], 4, 1, 128, 16),
    "prompt, heads of 256": ([(200, 100), (3, 7)], 4, 2, 256, 16),
    "prompt, heads of 256, splits": ([(1500, 100)], 4, 2, 256, 32),
    "prompts and single tokens": ([(900, 1), (300, 100), (5000, 1)], 8, 2, 128, 16),
}


def spoiled(b, seed):
    """(token, head, sees a key) of some rows: the first and last of each sequence among them."""
    g = torch.Generator().manual_seed(seed)
    rows, at = [], 0
    for n, m in b.lens:
        for i in sorted({0, m - 1, int(torch.randint(0, m, (1,), generator=g))}):
            rows.append((at + i, int(torch.randint(0, b.hq, (1,), generator=g)), n - m + i >= 0 and n > 0))
        at += m
    return rows


def compare(b, attn, rows, clean, lse_of_seen):  # noqa: F811
    got, lse = b.call(attn, return_lse=True)
    b.q = clean
    fine, fine_lse = b.call(attn, return_lse=True)
    for token, head, sees in rows:
        if sees:
            assert bool(got[token, head].isnan().all()), (token, head, got[token, head])
            assert lse_of_seen(lse[token, head].item()), (token, head, lse[token, head])
        else:
            assert bool((got[token, head] == 0).all()) and lse[token, head].item() == -float("inf")
        got[token, head], lse[token, head] = fine[token, head], fine_lse[token, head]
    b.check(got, lse)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("cut", CUTS)
def test_nan_in_a_query(attn, cut, dtype):  # noqa: F811
    b = Batch(*CUTS[cut], dtype, seed=11)
    clean, rows = b.q, spoiled(b, 1)
    b.q = clean.clone()
    for i, (token, head, _) in enumerate(rows):
        if i % 2:
            b.q[token, head] = float("nan")
        else:
            b.q[token, head, (7 * i) % b.d] = float("nan")
    compare(b, attn, rows, clean, lambda x: x != x)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("cut", CUTS)
@pytest.mark.parametrize("sign", [1, -1])
def test_infinity_in_a_query(attn, cut, sign, dtype):  # noqa: F811
    """Element 5 of every key is positive, so that all scores of a row with an infinity there are infinite of one
    sign: the weights are 0 / 0 either way, and the sum of the exponentials infinite or 0."""
    b = Batch(*CUTS[cut], dtype, seed=12)
    b.codes[:, 0, :, :, 2] = (b.codes[:, 0, :, :, 2] & 0x0F) | 0x20
    clean, rows = b.q, spoiled(b, 2)
    b.q = clean.clone()
    for token, head, _ in rows:
        b.q[token, head, 5] = sign * float("inf")
    # +: the logarithm of an infinite sum is infinite, or NaN where the sum was formed after the maximum was taken off
    compare(b, attn, rows, clean, (lambda x: x != x or x == float("inf")) if sign > 0 else (lambda x: x == -float("inf")))


@pytest.mark.parametrize("lens", [[(700, 1)], [(300, 200)], [(90, 1)]])
def test_a_position_outside_the_table_stays_marked(attn, lens):  # noqa: F811
    """The cache write answers such a position with a query of NaN; the attention behind it says so too."""
    from test_speed_scalesweep_b200 import kv_cache
    b = Batch(lens, 4, 2, 128, 16, "bf16", seed=13)
    t = b.q.shape[0]
    table, pos = kv_cache.rotary_cos_sin_cache(1000, 128), torch.arange(t, device="cuda")
    pos[-1] = 1000
    kv = torch.zeros(t, 2, 128, dtype=b.dtype, device="cuda")
    nowhere = torch.full((t,), -1, dtype=torch.int64, device="cuda")
    b.q = kv_cache.rotary_scalesweep_mse_nvfp4_kv_write(b.q, kv, kv, pos, table, nowhere, b.mult, b.codes, b.scales)
    out = b.call(attn)
    assert bool(out[-1].isnan().all()) and bool(out[:-1].isfinite().all())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("scale", [30.0, 1e6, 1e30])
@pytest.mark.parametrize("cut", CUTS)
def test_scores_past_what_float32_resolves_are_not_taken_for_no_key(attn, cut, scale, dtype):  # noqa: F811
    """Where neighbouring float32 scores lie further apart than softmax can weigh, a row may be NaN, but not zero:
    it saw keys, and their values are not 0."""
    b = Batch(*CUTS[cut], dtype, seed=14, spread=3e3)
    b.mult.fill_(1.0)
    b.codes[:, 1] = (b.codes[:, 1] & 0x77) | 0x11  # values of at least 0.5 times their scale
    out = b.call(attn, softmax_scale=scale)
    at = 0
    for n, m in b.lens:
        for i in range(m):
            none = n - m + i < 0 or n == 0
            assert bool((out[at + i] == 0).all()) if none else not bool((out[at + i] == 0).any()), (at + i, none)
        at += m
