"""Tangents: the operators have no forward-mode derivative and say so, instead of an answer without one."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _case():
    import imageni2r_amd as i2r
    gen = torch.Generator(DEV).manual_seed(0)
    q, k, v = (torch.randn(10, 2, 16, generator=gen, device=DEV) for _ in range(3))
    buckets = i2r.RelativeBuckets(8, 20)
    seqs = i2r.PackedSequences.from_lengths([4, 6], buckets=buckets)
    return [q, k, v, torch.randn(2, 8, generator=gen, device=DEV)], seqs, buckets


@pytest.mark.parametrize("at", range(4))
@pytest.mark.parametrize("grad", [True, False])
def test_packed_attention_refuses_a_tangent(at, grad):
    import imageni2r_amd as i2r
    ops, seqs, _ = _case()
    with fwad.dual_level(), torch.set_grad_enabled(grad):
        plain = i2r.packed_attention(*ops[:3], seqs, bias=ops[3])  # a level alone changes nothing
        ops[at] = fwad.make_dual(ops[at], torch.ones_like(ops[at]))
        with pytest.raises(RuntimeError, match="forward"):
            i2r.packed_attention(*ops[:3], seqs, bias=ops[3])
        with pytest.raises(ValueError, match="out="):
            i2r.packed_attention(*ops[:3], seqs, bias=ops[3], out=torch.empty_like(plain))


@pytest.mark.parametrize("grad", [True, False])
def test_relative_bias_refuses_a_tangent(grad):
    import imageni2r_amd as i2r
    ops, _, buckets = _case()
    with fwad.dual_level(), torch.set_grad_enabled(grad):
        i2r.relative_bias(ops[3], buckets, 5, 7)
        with pytest.raises(RuntimeError, match="forward"):
            i2r.relative_bias(fwad.make_dual(ops[3], torch.ones_like(ops[3])), buckets, 5, 7)
