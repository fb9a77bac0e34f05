"""The bias table's gradient beside keys and values that no query sees and that are not finite: hidden by -inf buckets or by a
score of -inf, with the last queries of a tile missing, by places and by given positions."""
import math

import pytest
import torch

from tests.packed_reference import check, reference

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.float16, torch.bfloat16]
BAD = [(math.nan, math.nan), (math.inf, -math.inf), (1.0, math.nan), (math.nan, 1.0)]


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _grads(q, k, v, table, seqs, dout):
    import imageni2r_amd as i2r
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v, table)]
    out = i2r.packed_attention(*leaves[:3], seqs, bias=leaves[3])
    return dict(zip(("out", "dq", "dk", "dv", "dtable"), (out.detach(),) + torch.autograd.grad(out, leaves, dout)))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("bad", BAD, ids=str)
@pytest.mark.parametrize("dim,heads,kv", [(8, 3, 3), (64, 4, 2), (128, 2, 1)])
@pytest.mark.parametrize("lq", [8, 40, 100])
@pytest.mark.parametrize("positions", [False, True], ids=["places", "positions"])
def test_buckets_that_hide(dtype, bad, dim, heads, kv, lq, positions):
    """Two sequences of lq queries at the end of more keys; distances of 64 and more are hidden, and so keys far before
    every query: what they hold reaches no gradient."""
    import imageni2r_amd as i2r
    gen = torch.Generator(DEV).manual_seed(dim + lq)
    rand = lambda *s: torch.randn(*s, generator=gen, device=DEV).to(dtype)
    lk = lq + 200
    cu_q, cu_k = [0, lq, 2 * lq], [0, lk, 2 * lk]
    q, dout, k, v = rand(2 * lq, heads, dim), rand(2 * lq, heads, dim), rand(2 * lk, kv, dim), rand(2 * lk, kv, dim)
    buckets = i2r.RelativeBuckets(16, 64, False)
    table = torch.randn(heads, 16, generator=gen, device=DEV)
    table[:, 15] = -math.inf
    pos = {}
    if positions:  # (places 0 and around, which no query holds, are near the hidden keys)
        pos = dict(pos_q=(torch.arange(2 * lq, device=DEV) % lq + 200).int(), pos_k=(torch.arange(2 * lk, device=DEV) % lk).int())
    seqs = i2r.PackedSequences(_i32(cu_q), _i32(cu_k), causal=True, buckets=buckets, **pos)
    ref = dict(cu_q=cu_q, cu_k=cu_k, causal=True, table=table, buckets=buckets, **pos)
    for at in (0, 5, 100, 130, 136, lk + 1, lk + 131, lk + 136):
        k[at], v[at] = bad
    want = reference(q, k, v, dout=dout, **ref)
    assert all(bool(torch.isfinite(w[0]).all()) for w in want.values())
    got = _grads(q, k, v, table, seqs, dout)
    for name, w in want.items():
        check(name, got[name], *w)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim", [8, 64, 128])
@pytest.mark.parametrize("lq", [1, 32, 45])
def test_scores_that_hide(dtype, dim, lq):
    """Keys whose product with every query is -inf are hidden, NaN in their values: the gradients are those without them."""
    import imageni2r_amd as i2r
    gen = torch.Generator(DEV).manual_seed(dim + lq)
    rand = lambda *s: torch.randn(*s, generator=gen, device=DEV).to(dtype)
    lk, gone = 150, [3, 70, 149]
    q, dout, k, v = rand(lq, 2, dim), rand(lq, 2, dim), rand(lk, 2, dim), rand(lk, 2, dim)
    q[..., 0] = -1.0
    table = torch.randn(2, 16, generator=gen, device=DEV)
    buckets = i2r.RelativeBuckets(16, 64, True)
    pos_q = torch.randint(0, 200, (lq,), generator=gen, device=DEV).int()
    pos_k = torch.randint(0, 200, (lk,), generator=gen, device=DEV).int()
    keep = torch.ones(lk, dtype=torch.bool, device=DEV)
    keep[gone] = False
    want = reference(q, k[keep], v[keep], [0, lq], [0, lk - 3], table=table, buckets=buckets, pos_q=pos_q, pos_k=pos_k[keep],
                     dout=dout)
    k[gone, :, 0], v[gone] = math.inf, math.nan
    seqs = i2r.PackedSequences(_i32([0, lq]), _i32([0, lk]), buckets=buckets, pos_q=pos_q, pos_k=pos_k)
    got = _grads(q, k, v, table, seqs, dout)
    for name, w in want.items():
        check(name, got[name][keep] if name in ("dk", "dv") else got[name], *w)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim", [8, 64, 128])
def test_a_value_that_is_seen_stays_in_its_buckets(dtype, dim):
    """A NaN in one query's output gradient is in the buckets of the pairs that it sees, and in no other's sum; beside it the
    sums are those of the other queries to the bit of the formula."""
    import imageni2r_amd as i2r
    gen = torch.Generator(DEV).manual_seed(dim)
    rand = lambda *s: torch.randn(*s, generator=gen, device=DEV).to(dtype)
    n, row = 50, 7
    q, k, v, dout = (rand(n, 2, dim) for _ in range(4))
    buckets = i2r.RelativeBuckets(16, 64, False)
    table = torch.randn(2, 16, generator=gen, device=DEV)
    seqs = i2r.PackedSequences(_i32([0, n]), causal=True, buckets=buckets)
    want = reference(q, k, v, [0, n], causal=True, table=table, buckets=buckets, dout=dout)
    dout[row, 1] = math.nan
    got = _grads(q, k, v, table, seqs, dout)["dtable"]
    reached = buckets.bucket(torch.arange(row + 1, device=DEV) - row)
    hit = torch.zeros(2, 16, dtype=torch.bool, device=DEV)
    hit[1, reached] = True
    assert torch.equal(torch.isnan(got), hit)
    check("dtable", got[~hit], want["dtable"][0][~hit], want["dtable"][1][~hit])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_captured(dtype):
    """A replayed backward whose keys turn NaN and finite again: every replay has the eager call's bits."""
    import imageni2r_amd as i2r
    from imageni2r_amd import packed
    gen = torch.Generator(DEV).manual_seed(1)
    rand = lambda *s: torch.randn(*s, generator=gen, device=DEV).to(dtype)
    q, dout, k, v = rand(40, 2, 64), rand(40, 2, 64), rand(240, 2, 64), rand(240, 2, 64)
    buckets = i2r.RelativeBuckets(16, 64, False)
    table = torch.randn(2, 16, generator=gen, device=DEV)
    table[:, 15] = -math.inf
    seqs = i2r.PackedSequences(_i32([0, 40]), _i32([0, 240]), causal=True, buckets=buckets)

    def step():
        out, out32, stats = packed.packed_attention_fwd(q, k, v, seqs, table, save=True)
        return (out,) + packed.packed_attention_bwd(q, k, v, seqs, table, out32, stats, dout)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for value in (math.nan, 0.5, math.inf, math.nan, -1.0):
        k[130], v[130] = value, value
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(bool(torch.isfinite(t).all()) for t in want)
        assert all(torch.equal(a, b) for a, b in zip(held, want))
