"""The completion stage's encoder on packed sequences: the same values and gradients as torch's padded encoder, with the
bias of `relative_bias` as its additive mask; and the train iteration around it."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _models(buckets, dropout=0.0):
    from imageni2r_amd.tst_boundary import CompletionStandIn
    torch.manual_seed(0)
    padded = CompletionStandIn(7, 96, num_layers=3, dim_feedforward=64, dropout=dropout).to(DEV)
    torch.manual_seed(0)
    packed = CompletionStandIn(7, 96, num_layers=3, dim_feedforward=64, dropout=dropout, packed=True, rel_buckets=buckets,
                               rel_distance=40).to(DEV)
    missing = packed.load_state_dict(padded.state_dict(), strict=False)
    assert not missing.unexpected_keys and missing.missing_keys == (["rel_bias"] if buckets else [])
    return padded, packed


def _batch(B=6, L=96, C=7):
    gen = torch.Generator().manual_seed(5)
    x = torch.rand(B, L, C, generator=gen)
    for b in range(B):
        x[b, torch.randperm(L, generator=gen)[: 10 + 15 * b]] = float("nan")
    return x.to(DEV)


def _padded_embed(m, x, mask, bias):
    """CompletionStandIn.embed in 64 bits, the bias and the hidden keys as torch's additive mask."""
    z = torch.nan_to_num(x.double(), nan=0.0)
    z = m.project_inp(z) * m.d_model**0.5 + m.pe[:, : z.shape[1]]
    hide = torch.zeros(mask.shape, dtype=torch.float64, device=DEV).masked_fill_(~mask, float("-inf"))
    add = (bias.double()[None] + hide[:, None, None, :]).reshape(-1, z.shape[1], z.shape[1])
    return m.output_layer(torch.nn.functional.gelu(m.encoder(z, mask=add)))


@pytest.mark.parametrize("buckets", [0, 16])
def test_packed_encoder_is_the_padded_encoder(buckets):
    """Against 64 bits.  fp32: 3 layers of sums of at most 96 terms between layer norms; 2^-24 times a few hundred roundings
    is 3e-5 of the values' size."""
    from imageni2r_amd import relative_bias
    padded, packed = _models(buckets)
    x = _batch()
    mask = ~torch.isnan(x).any(-1)
    dense = torch.zeros(5, 96, 96, device=DEV)
    if buckets:
        torch.nn.init.normal_(packed.rel_bias, generator=torch.Generator(DEV).manual_seed(1))
        table = packed.rel_bias.detach().clone().requires_grad_(True)
        dense = relative_bias(table, packed.buckets, 96, 96)
    exact = copy.deepcopy(padded).double()
    exact.train()  # (dropout 0: training mode only keeps torch off its fused inference path)
    want = _padded_embed(exact, x, mask, dense)
    got = packed.embed(x, mask)
    weight = torch.randn(got.shape, generator=torch.Generator(DEV).manual_seed(2), device=DEV)
    assert float((got.double() - want).abs().max()) <= 3e-5 * float(want.abs().max())
    (got * weight).sum().backward()
    (want * weight.double()).sum().backward()
    exact_grads = dict(exact.named_parameters())
    for name, p in packed.named_parameters():
        if p.grad is None:
            continue
        ref = table.grad.double() if name == "rel_bias" else exact_grads[name].grad
        assert float((p.grad.double() - ref).norm()) <= 1e-4 * float(ref.norm()), name
    assert not buckets or packed.rel_bias.grad is not None


def test_a_series_without_observed_steps_is_finite():
    _, packed = _models(16)
    x = _batch()
    x[2] = float("nan")
    out = packed(x, ~torch.isnan(x).any(-1))
    out.sum().backward()
    assert bool(torch.isfinite(out).all()) and all(bool(torch.isfinite(p.grad).all()) for p in packed.parameters())


def test_train_iteration_with_a_packed_completion():
    """Two iterations around a replayed diffusion step: losses finite, every completion weight (the bias too) moves, and
    the recovery loss is what the packed model gives on its own."""
    from imageni2r_amd import FusedAdamW, GraphedTrainStep, TS2img_Karras
    from imageni2r_amd.tst_boundary import CompletionStandIn, TrainIteration, recovery_loss
    from tests.helpers import tiny_args
    torch.manual_seed(0)
    a = tiny_args(device=DEV)
    model = TS2img_Karras(a, DEV).to(DEV)
    comp = CompletionStandIn(3, 24, num_layers=2, dim_feedforward=64, dropout=0.0, packed=True, rel_buckets=8,
                             rel_distance=12).to(DEV)
    it = TrainIteration(model, comp, torch.optim.AdamW(comp.parameters(), lr=1e-3),
                        diffusion_step=GraphedTrainStep(model, FusedAdamW(model.net.parameters(), lr=1e-4, max_grad_norm=1.0)))
    gen = torch.Generator().manual_seed(3)
    x = torch.rand(4, 24, 3, generator=gen)
    x[:, 5:9], x[1, 12:20] = float("nan"), float("nan")
    x = x.to(DEV)
    before = [p.detach().clone() for p in comp.parameters()]
    with torch.no_grad():
        alone = recovery_loss(comp(x, ~torch.isnan(x).any(-1)), x)
    for n in range(2):
        loss, loss_e = it(x.clone())
        assert torch.isfinite(loss) and torch.isfinite(loss_e)
        if n == 0:
            assert abs(loss_e.item() - alone.item()) <= 1e-5 * abs(alone.item())
    assert all(not torch.equal(a, b.detach()) for a, b in zip(before, comp.parameters()))
