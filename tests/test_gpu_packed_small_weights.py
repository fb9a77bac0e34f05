"""Probabilities far below fp16's smallest numbers that count together: one key far above many others."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("rows", [1, 40, 200])
@pytest.mark.parametrize("keys", [300, 4096, 20000])
@pytest.mark.parametrize("dim", [8, 64, 128])
@pytest.mark.parametrize("bias", [False, True], ids=["plain", "bias"])
def test_many_small_beside_a_large_one(rows, keys, dim, bias):
    """Key 0 has score 0 and value 0, the others -17.5 and 64: the output is 64 s / (1 + s), s = (keys - 1) e^-17.5, though
    each probability, 2^-25.2, rounds to 0 in fp16.

    Held 2^7 times as large, each is off by at most half of fp16's smallest step, 2^-25 / 2^7 = 2^-32; the sums over the keys
    by 2^-24 a key; the output by half a step of its own, 2^-11, and of fp16's smallest."""
    import imageni2r_amd as i2r
    from imageni2r_amd import packed
    q = torch.zeros(rows, 4, dim, device=DEV, dtype=torch.float16)
    k = torch.zeros(keys, 2, dim, device=DEV, dtype=torch.float16)
    v = torch.full((keys, 2, dim), 64.0, device=DEV, dtype=torch.float16)
    q[..., 0], k[1:, :, 0], v[0] = 1.0, -17.5, 0.0
    buckets = i2r.RelativeBuckets(8, 20) if bias else None
    table = torch.zeros(4, 8, device=DEV) if bias else None
    ends = [torch.tensor([0, n], dtype=torch.int32, device=DEV) for n in (rows, keys)]
    seqs = i2r.PackedSequences(*ends, buckets=buckets)
    s = (keys - 1) * torch.tensor(-17.5, dtype=torch.float64).exp().item()
    want = 64.0 * s / (1.0 + s)
    sums = 64.0 * keys * 2.0**-32 + want * (keys + 64) * 2.0**-24
    if not bias:  # (with a bias to train the second term of each probability leaves 2^-32 again; without, fp16's half step)
        sums += want * 2.0**-11
    out, out32, _ = packed.packed_attention_fwd(q, k, v, seqs, table, 1.0, save=True)
    assert float((out32.double() - want).abs().max()) <= sums
    bound = sums + want * 2.0**-11 + 2.0**-25
    assert float((out.double() - want).abs().max()) <= bound
    got = i2r.packed_attention(q, k, v, seqs, bias=table, scale=1.0)
    assert float((got.double() - want).abs().max()) <= bound + want * 2.0**-11


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("rows,keys", [(1, 2000), (1, 40), (150, 300)])
@pytest.mark.parametrize("size", [0.0, 1e3, 2.0**25, 2.0**26, 2.0**27, 1e38])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("bias", [False, True], ids=["plain", "bias"])
def test_equal_scores_of_any_size(dtype, rows, keys, size, sign, bias):
    """Keys that are all alike weigh alike, also where the scores are so large that 7 is less than their last place: the mean of
    the values, off by half a step of the type for each probability and once more for the output, and 2^-24 a key.  The table's
    lowest value, -3.4e38, and a product of -1e38 are -4.4e38 together, in 32 bits -inf: such keys are hidden, the output is 0."""
    import imageni2r_amd as i2r
    gen = torch.Generator(DEV).manual_seed(keys)
    q = torch.ones(rows, 2, 8, device=DEV, dtype=dtype)
    k = torch.ones(keys, 1, 8, device=DEV, dtype=dtype)
    v = torch.randn(keys, 1, 8, generator=gen, device=DEV).to(dtype)
    hidden = bias and size == 1e38 and sign < 0
    table = torch.full((2, 8), torch.finfo(torch.float32).min if hidden else 0.0, device=DEV) if bias else None
    ends = [torch.tensor([0, n], dtype=torch.int32, device=DEV) for n in (rows, keys)]
    seqs = i2r.PackedSequences(*ends, buckets=i2r.RelativeBuckets(8, 20) if bias else None)
    u = torch.finfo(dtype).eps / 2
    want = v.double().mean(0) * (not hidden)
    bound = 2 * u * want.abs() + (u + (keys + 16) * 2.0**-24) * v.double().abs().mean(0)
    got = i2r.packed_attention(q, k, v, seqs, bias=table, scale=sign * size / 8)
    assert bool(((got.double() - want).abs() <= bound).all())
    leaf = table.requires_grad_(True) if bias else q.requires_grad_(True)  # (what a backward pass needs is kept: another form)
    got = i2r.packed_attention(q, k, v, seqs, bias=table, scale=sign * size / 8)
    assert leaf.requires_grad and bool(((got.detach().double() - want).abs() <= bound).all())


@pytest.mark.parametrize("rows,keys,heads,kv", [(1, 2000, 4, 2), (3, 40, 4, 4), (90, 300, 4, 1)])
@pytest.mark.parametrize("dim", [16, 64, 128])
@pytest.mark.parametrize("lowest", ["all", "far", "near"])
def test_fp16_tables_of_the_lowest_value(rows, keys, heads, kv, dim, lowest):
    """Buckets of the type's lowest value in fp16, where the exponent that 2^7 is taken from has no place left for it: rows that
    have nothing else weigh their keys alike, others leave those keys out; with gradients."""
    import imageni2r_amd as i2r
    from tests.packed_reference import check, reference
    gen = torch.Generator(DEV).manual_seed(dim + rows)
    q, dout = (torch.randn(rows, heads, dim, generator=gen, device=DEV).half() for _ in range(2))
    k, v = (torch.randn(keys, kv, dim, generator=gen, device=DEV).half() for _ in range(2))
    buckets = i2r.RelativeBuckets(16, 40, False)
    table = torch.randn(heads, 16, generator=gen, device=DEV)
    table[:, {"all": slice(None), "far": slice(15, 16), "near": slice(0, 15)}[lowest]] = torch.finfo(torch.float32).min
    seqs = i2r.PackedSequences(torch.tensor([0, rows], dtype=torch.int32, device=DEV),
                               torch.tensor([0, keys], dtype=torch.int32, device=DEV), causal=True, buckets=buckets)
    want = reference(q, k, v, [0, rows], [0, keys], causal=True, table=table, buckets=buckets, dout=dout)
    with torch.no_grad():
        check("out, inference", i2r.packed_attention(q, k, v, seqs, bias=table), *want["out"])
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v, table)]
    out = i2r.packed_attention(*leaves[:3], seqs, bias=leaves[3])
    got = dict(zip(("out", "dq", "dk", "dv", "dtable"), (out.detach(),) + torch.autograd.grad(out, leaves, dout)))
    for name, w in want.items():
        check(name, got[name], *w)
