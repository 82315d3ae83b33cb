"""GPU checks that the cache's operators, which have no backward pass, refuse
inputs whose gradients they would drop."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from test_gpu_kv_attention import Batch, attn  # noqa: F401  (attn: the fixture)

pytestmark = pytest.mark.gpu


def calls(attn):  # noqa: F811
    """Each operator as a function of its floating inputs, and those inputs."""
    from test_speed_scalesweep_b200 import kv_cache, ops  # noqa: F401
    b = Batch([(40, 5)], 4, 2, 64, 16, "bf16", seed=41)
    kv = torch.randn(2, 5, 2, 64, device="cuda").bfloat16()
    idx, table = torch.arange(5, device="cuda"), kv_cache.rotary_cos_sin_cache(16, 64)
    ns = torch.ops.scalesweep_b200

    def write(q, k, v, t, mult):
        return kv_cache.rotary_scalesweep_mse_nvfp4_kv_write(q, k, v, idx, t, idx, mult, b.codes, b.scales)

    def write_op(q, k, v, t, mult):
        return ns.rotary_scalesweep_mse_nvfp4_kv_write(q, k, v, idx, t, idx, mult, b.codes, b.scales)

    def write_into(out):
        return kv_cache.rotary_scalesweep_mse_nvfp4_kv_write(b.q, kv[0], kv[1], idx, table, idx, b.mult, b.codes,
                                                             b.scales, query_out=out)

    def attend(q, mult):
        return attn.nvfp4_paged_attention(q, b.codes, b.scales, mult, b.table, b.seq_lens, b.start, 5, 40)

    def attend_op(q, mult):
        return ns.nvfp4_paged_attention(q, b.codes, b.scales, mult, b.table, b.seq_lens, b.start, 5, 40)

    def attend_into(out):
        return attn.nvfp4_paged_attention(b.q, b.codes, b.scales, b.mult, b.table, b.seq_lens, b.start, 5, 40, out=out)

    def gather(mult):
        return kv_cache.nvfp4_kv_gather(b.codes, b.scales, mult, idx)[0]
    w = (b.q, kv[0], kv[1], table, b.mult)
    return [(write, w), (write_op, w), (write_into, (b.q,)), (attend, (b.q, b.mult)), (attend_op, (b.q, b.mult)),
            (attend_into, (b.q,)), (gather, (b.mult,))]


def test_inputs_that_require_a_gradient_are_refused(attn):  # noqa: F811
    for f, inputs in calls(attn):
        for i in range(len(inputs)):
            args = [t.clone().requires_grad_(j == i) for j, t in enumerate(inputs)]
            with pytest.raises(ValueError, match="gradient"):
                f(*args)
            with torch.no_grad():
                want = f(*args)
            with torch.inference_mode():
                assert torch.equal(f(*args), want)
            assert not want.requires_grad or want is args[i]


def test_forward_mode_is_refused(attn):  # noqa: F811
    for f, inputs in calls(attn):
        for i in range(len(inputs)):
            with fwd.dual_level():
                args = [fwd.make_dual(t.clone(), torch.ones_like(t)) if j == i else t for j, t in enumerate(inputs)]
                with pytest.raises(ValueError, match="forward-mode"):
                    f(*args)


def test_wrapped_tensors_are_refused(attn):  # noqa: F811
    for f, inputs in calls(attn):
        if f.__name__.endswith("op"):
            continue  # the dispatcher's own rules
        stacked = torch.stack([inputs[0]] * 2)
        with pytest.raises((ValueError, RuntimeError)):
            torch.vmap(lambda x: f(x, *inputs[1:]))(stacked)
