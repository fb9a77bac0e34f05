"""The dense relative position bias (imageni2r_amd.relative_bias) and its table's gradient."""
import pytest
import torch

from tests.packed_reference import bucket_by_logarithms

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _case(gen, heads, nq, nk, bias, positions):
    import imageni2r_amd as i2r
    table = torch.randn(heads, bias[0], generator=gen, device=DEV)
    pos = (None, None)
    if positions:
        pos = tuple(torch.randint(-2**31, 2**31 - 1, (n,), generator=gen, device=DEV).int() if positions == "any" else
                    torch.randint(0, 200, (n,), generator=gen, device=DEV).int() for n in (nq, nk))
    pq, pk = (torch.arange(nk - nq, nk, device=DEV), torch.arange(nk, device=DEV)) if not positions else \
        (pos[0].long(), pos[1].long())
    bucket = bucket_by_logarithms(pk[None, :] - pq[:, None], *bias)
    return i2r.RelativeBuckets(*bias), table, pos, bucket


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("heads,nq,nk", [(1, 1, 1), (5, 96, 96), (3, 1, 777), (7, 130, 65), (16, 33, 1000), (70, 9, 24),
                                         (2, 515, 3)])
@pytest.mark.parametrize("bias", [(32, 128, True), (64, 1024, True), (7, 30, False)], ids=str)
@pytest.mark.parametrize("positions", [None, "near", "any"])
def test_bias_and_gradient(dtype, heads, nq, nk, bias, positions):
    import imageni2r_amd as i2r
    gen = torch.Generator(DEV).manual_seed(nq + nk)
    buckets, table, pos, bucket = _case(gen, heads, nq, nk, bias, positions)
    table.requires_grad_(True)
    out = i2r.relative_bias(table, buckets, nq, nk, *pos, dtype=dtype)
    assert torch.equal(out, table.detach()[:, bucket].to(dtype))
    dout = torch.randn(heads, nq, nk, generator=gen, device=DEV).to(dtype)
    (got,) = torch.autograd.grad(out, table, dout)
    flat, d = bucket.reshape(-1), dout.double().reshape(heads, -1)
    want = torch.zeros(heads, bias[0], dtype=torch.float64, device=DEV).index_add_(1, flat, d)
    size = torch.zeros_like(want).index_add_(1, flat, d.abs())
    # fp32 sums of fp32 terms: each of the at most nq * nk / 64 + 64 partial sums a term passes through rounds once
    bound = (nq * nk / 64 + 64) * 2.0**-24 * size
    assert bool(((got.double() - want).abs() <= bound).all())
    with torch.no_grad():
        assert torch.equal(i2r.relative_bias(table, buckets, nq, nk, *pos, dtype=dtype), out)


def test_large_and_repeated():
    import imageni2r_amd as i2r
    gen = torch.Generator(DEV).manual_seed(0)
    buckets, table, pos, bucket = _case(gen, 12, 1501, 2047, (32, 128, True), None)
    dout = torch.randn(12, 1501, 2047, generator=gen, device=DEV)
    table.requires_grad_(True)
    got = [torch.autograd.grad(i2r.relative_bias(table, buckets, 1501, 2047), table, dout)[0] for _ in range(3)]
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
    want = torch.zeros(12, 32, dtype=torch.float64, device=DEV).index_add_(1, bucket.reshape(-1), dout.double().reshape(12, -1))
    assert float((got[0].double() - want).norm() / want.norm()) < 2e-6  # 3e6 terms: random roundings of 2^-24


def test_special_values_stay_in_their_bucket():
    import imageni2r_amd as i2r
    gen = torch.Generator(DEV).manual_seed(0)
    buckets, table, pos, bucket = _case(gen, 2, 70, 90, (8, 20, False), None)
    table[0, 3], table[1, 2], table[0, 1] = float("-inf"), float("nan"), torch.finfo(torch.float32).min
    out = i2r.relative_bias(table, buckets, 70, 90)
    assert torch.equal(torch.nan_to_num(out, 7.0), torch.nan_to_num(table[:, bucket], 7.0))
    dout = torch.randn(2, 70, 90, generator=gen, device=DEV)
    clean = i2r.packed.relative_bias_bwd(dout, buckets)
    dout[0][bucket == 5] = float("nan")
    got = i2r.packed.relative_bias_bwd(dout, buckets)
    assert bool(torch.isnan(got[0, 5])) and torch.equal(got[1], clean[1])
    keep = torch.arange(8, device=DEV) != 5
    assert torch.equal(got[0][keep], clean[0][keep])


def test_no_places():
    import imageni2r_amd as i2r
    buckets = i2r.RelativeBuckets(8, 20)
    for n in ((0, 5), (5, 0), (0, 0)):
        t = torch.ones(3, 8, device=DEV, requires_grad=True)
        out = i2r.relative_bias(t, buckets, *n)
        assert out.shape == (3, *n)
        assert bool((torch.autograd.grad(out, t, out.detach())[0] == 0).all())


def test_captured_gradient_replays():
    import imageni2r_amd as i2r
    from imageni2r_amd import packed
    gen = torch.Generator(DEV).manual_seed(0)
    buckets, table, pos, bucket = _case(gen, 4, 300, 200, (32, 64, True), "near")
    dout = torch.randn(4, 300, 200, generator=gen, device=DEV)
    f = lambda: (packed.relative_bias_fwd(table, buckets, 300, 200, *pos), packed.relative_bias_bwd(dout, buckets, *pos))
    f()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = f()
    for _ in range(3):
        table.normal_(generator=gen)
        dout.normal_(generator=gen)
        want = f()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals():
    import imageni2r_amd as i2r
    t = torch.ones(3, 8, device=DEV)
    b = i2r.RelativeBuckets(8, 20)
    pos = torch.zeros(5, dtype=torch.int32, device=DEV)
    for bad, kind in ((dict(table=t[:, :4]), ValueError), (dict(table=t.half()), TypeError), (dict(q_len=-1), ValueError),
                      (dict(table=t.cpu()), i2r.ops._lib.I2RError), (dict(buckets=None), TypeError), (dict(pos_q=pos), ValueError),
                      (dict(pos_q=pos, pos_k=pos), ValueError), (dict(pos_q=pos.long(), pos_k=pos.long()), TypeError),
                      (dict(dtype=torch.float64), TypeError)):
        with pytest.raises(kind):
            i2r.relative_bias(**{**dict(table=t, buckets=b, q_len=5, k_len=6), **bad})
